// Paged cache: what the kernels and the C ABI share (layout, batch of sequences, launch interface).
//
// K and V: [layer][page][kv_head][slot][d].  Position j of sequence s is slot j % page_size of page table[s][j / page_size]; the
// page size is a power of two.  Lengths, offsets and page numbers come from device arrays that the host has not seen, so the
// kernels bound every one of them before it becomes an address.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace vfkv {

constexpr uint32_t kPagedMaxLen = 1u << 23;   // positions of one sequence: the 16-key units of a whole batch are counted in 32 bits

struct PagedSlab {             // one layer
    const uint8_t* k;
    const uint8_t* v;
    uint64_t page_bytes;       // one page of one layer, one tensor
    uint32_t n_pages, page_shift, n_kv_heads, head_dim, dtype;
};
struct PagedSeqs {
    const int32_t* table;      // [n_seqs][table_stride]
    const int32_t* kv_lens;    // [n_seqs]
    const int32_t* q_offsets;  // [n_seqs + 1] or NULL: token t is the one token of sequence t
    uint32_t n_seqs, table_stride, n_tokens;
    uint32_t limit;            // min(table_stride * page_size, kPagedMaxLen): positions from here on have no row
};
struct PagedAttnLaunch {
    PagedSlab c;
    PagedSeqs s;
    const void* q = nullptr;
    void* o = nullptr;
    uint64_t q_stride = 0, o_stride = 0;   // elements between two tokens
    uint32_t n_heads = 0, window = 0, n_sink = 0;
    uint32_t io_f16 = 0;                   // q and o are f16 (else f32)
    uint32_t max_kv = 0;                   // upper bound of the lengths that the host knows
    float scale = 0.f, softcap = 0.f;
    float* scratch_out = nullptr;          // partial outputs, maxima and sums of the parts of a sequence
    float* scratch_max = nullptr;
    float* scratch_sum = nullptr;
    uint64_t scratch_rows = 0;             // partial rows (of head_dim floats) the scratch holds
};
struct PagedWriteLaunch {
    PagedSlab c;
    PagedSeqs s;
    const void* q; const float* q_weight; void* q_out;
    const void* k; const void* v; const float* k_weight;
    const int32_t* positions; const float* freq_factors;
    uint64_t q_stride, q_out_stride, k_stride, v_stride;
    uint32_t n_heads, io_f16;
    uint32_t mode, rotary_dim, n_axes, interleaved, section[4];
    double log2_step;                      // log2 of the frequency ratio of neighbouring pairs: -2 log2(base) / rotary_dim
    float freq_scale, attn_factor, eps;
};
constexpr uint32_t kPagedMaxSeqs = 4096;   // sequences per call: their unit counts are summed in LDS
constexpr uint32_t kCopyPairs = 256;       // page copies per launch: they travel as kernel arguments
struct PagedCopyLaunch {
    uint8_t* k;                            // whole buffers
    uint8_t* v;
    uint64_t layer_bytes, page_bytes;
    uint32_t n_layers, n_kv_heads, page_size, row_bytes;   // row_bytes: one slot of one KV head
    uint32_t n;
    const uint32_t* src; const uint32_t* dst; const uint32_t* rows;   // host arrays, n <= kCopyPairs; rows NULL = all
};

hipError_t launch_paged_copy(const PagedCopyLaunch& L, hipStream_t stream);
hipError_t launch_paged_write(const PagedWriteLaunch& L, hipStream_t stream);
// Matrix-core kernels: head_dim a multiple of 16 up to 512 (F32 pages: 256); q and o 16-byte aligned with strides that keep every row so.
hipError_t launch_paged_decode(const PagedAttnLaunch& L, hipStream_t stream);
hipError_t launch_paged_prefill(const PagedAttnLaunch& L, hipStream_t stream);
hipError_t launch_paged_prefill_full(const PagedAttnLaunch& L, hipStream_t stream);    // F32 pages
hipError_t launch_paged_prefill_half(const PagedAttnLaunch& L, hipStream_t stream);    // F16
hipError_t launch_paged_prefill_byte(const PagedAttnLaunch& L, hipStream_t stream);    // FP8
hipError_t launch_paged_rows_merge(const PagedAttnLaunch& L, uint32_t n_split, hipStream_t stream);
// Workgroups per head group (KV head and slice of its query heads) the decode launch may use: its scratch holds two partial
// rows per workgroup and head.
uint32_t paged_decode_wgs(uint32_t head_groups);
// One wavefront per (token, head): any head_dim <= 512, any alignment.
hipError_t launch_paged_generic(const PagedAttnLaunch& L, hipStream_t stream);

#ifdef __HIPCC__
// Running maximum of a row that has seen no key yet: below every score.
constexpr float kNoScore = -3.40282347e38f;
// Weights are 2^(score - running maximum - ...): a maximum is raised when a score passes it by 2^kRaise, and a raised row's largest weight
// is 2^kBias.  Over FP8 and F16 pages as large as f16 takes them (at most 2^14, smallest step 2^-30 of the largest).  Over F32 pages at
// most 2^-6: 2^23 of them sum to 2^17, so elements of V up to 2^110 stay finite under any number of keys.
constexpr float kRaise = 8.f;               // log2
template <uint32_t DT>
constexpr float kBias = DT == kF32 ? -14.f : 6.f;
// A row is far out when its maximum (log2 units) leaves [-2^24, 2^24]: score * factor rounded once for the maximum and left exact
// inside the multiply-add of a weight would differ by more than a unit of log2 there, and the weights leave their f16 range.
__device__ __forceinline__ bool paged_far(float m) { return fabsf(m) > 16777216.f && m != kNoScore; }
// Logit soft-cap in log2 units, cap * tanh(y / cap), to a few steps of f32 at every size: the truncated continued fraction of tanh
// (7 / 5 terms, 8e-9 relative) below 0.8, 1 - 2 / (exp(2 x) + 1) on the hardware exponential and reciprocal above.  (The second alone
// is off by 1e-7 absolute, which a cap of 50 turns into 5e-6 of a score.)
__device__ __forceinline__ float paged_softcap_l2(float y, float cap_l2, float inv_cap_l2) {
    const float x = fabsf(y * inv_cap_l2), a = x * x;
    const float near = x * __builtin_fmaf(a, a + 105.f, 945.f) * __builtin_amdgcn_rcpf(__builtin_fmaf(a, __builtin_fmaf(a, 15.f, 420.f), 945.f));
    const float t = __builtin_amdgcn_exp2f(x * 2.88539008177793f);       // exp(2 x)
    const float far = __builtin_fmaf(-2.0f, __builtin_amdgcn_rcpf(t + 1.0f), 1.0f);
    return copysignf(cap_l2 * (x < 0.8f ? near : far), y);
}
// Length of sequence s as given, not negative: what positions are counted from.  It may pass S.limit: positions from there on have no
// row, so whoever turns one into a table entry compares it first.
__device__ __forceinline__ uint32_t paged_kv_len(const PagedSeqs& S, uint32_t s) {
    const int32_t n = S.kv_lens[s];
    return n < 0 ? 0u : (uint32_t)n;
}
// Token rows [lo, hi) of sequence s.
__device__ __forceinline__ void paged_rows(const PagedSeqs& S, uint32_t s, uint32_t& lo, uint32_t& hi) {
    if (S.q_offsets == nullptr) { lo = s; hi = s + 1u; return; }
    const int32_t a = S.q_offsets[s], b = S.q_offsets[s + 1u];
    lo = a < 0 ? 0u : (uint32_t)a < S.n_tokens ? (uint32_t)a : S.n_tokens;
    hi = b < 0 ? 0u : (uint32_t)b < S.n_tokens ? (uint32_t)b : S.n_tokens;
    if (hi < lo) hi = lo;
}
// Sequence of token t (n_seqs when it has none): the first whose rows end behind t.
__device__ __forceinline__ uint32_t paged_seq_of(const PagedSeqs& S, uint32_t t) {
    if (S.q_offsets == nullptr) return t < S.n_seqs ? t : S.n_seqs;
    uint32_t a = 0u, b = S.n_seqs;
    while (a < b) {
        const uint32_t mid = (a + b) >> 1;
        if (S.q_offsets[mid + 1u] > (int32_t)t) b = mid; else a = mid + 1u;
    }
    return a < S.n_seqs && S.q_offsets[a] <= (int32_t)t ? a : S.n_seqs;
}
// Page of positions [i * page_size, (i + 1) * page_size) of sequence s; n_pages when there is none.
__device__ __forceinline__ uint32_t paged_page(const PagedSlab& c, const PagedSeqs& S, uint32_t s, uint32_t i) {
    const uint32_t p = (uint32_t)S.table[(uint64_t)s * S.table_stride + i];
    return p < c.n_pages ? p : c.n_pages;
}
// First key of the window of the query at position p (keys in front of it are visible only as one of the first n_sink).
__device__ __forceinline__ uint32_t paged_window_lo(uint32_t window, uint32_t p) { return window != 0u && p + 1u > window ? p + 1u - window : 0u; }
#endif

}  // namespace vfkv
