// Attention over the paged cache: the generic form.  (paged_decode.hip and paged_prefill.h hold the matrix-core kernels.)
#include "device_utils.h"
#include "paged.h"

namespace vfkv {

// ---- generic form --------------------------------------------------------------------------------
// One wavefront per (token, head), for the head widths and alignments the matrix-core kernels do not take.  64 keys at a time: a
// lane forms the whole score of one key, then the lanes share the value columns; running maximum and sum in f32.  Bound by the latency
// of its loads, so sixteen elements of a key and the columns of eight keys are requested at a time (one at a time: five times slower).  Decode, 4 sequences
// of 1 000 keys, 8 / 2 heads: rows of 72 0.11 ms, F32 rows of 512 0.57 ms.
template <typename T, int DT>
__global__ __launch_bounds__(256) void paged_generic_kernel(PagedAttnLaunch a) {
    __shared__ float q_lds[4][512];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const uint32_t tok = blockIdx.x, head = blockIdx.y * 4u + (uint32_t)w;
    const uint32_t s = paged_seq_of(a.s, tok);
    if (s >= a.s.n_seqs || head >= a.n_heads) return;
    uint32_t r0, r1;
    paged_rows(a.s, s, r0, r1);
    const int64_t pos = (int64_t)paged_kv_len(a.s, s) - (int64_t)(r1 - tok);
    const uint32_t D = a.c.head_dim, kvh = head / (a.n_heads / a.c.n_kv_heads);
    constexpr uint32_t es = DT == kF32 ? 4u : DT == kF16 ? 2u : 1u;
    float* const q = q_lds[w];
    for (uint32_t d = lane; d < D; d += kWave)
        q[d] = (float)reinterpret_cast<const T*>(a.q)[(uint64_t)tok * a.q_stride + (uint64_t)head * D + d] * a.scale;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    float m = kNoScore, l = 0.f;
    if (pos >= 0) {
        // keys up to the query's own, as far as the table has rows
        const uint32_t end = (uint32_t)pos < a.s.limit ? (uint32_t)pos + 1u : a.s.limit, wlo = paged_window_lo(a.window, (uint32_t)pos);
        const uint32_t lo = wlo < end ? wlo : end, sink = a.n_sink < lo ? a.n_sink : lo;
        // chunks of the first tokens, then chunks of the window
        const uint32_t nsc = (sink + 63u) / 64u, nwc = (end - lo + 63u) / 64u;
        for (uint32_t c = 0; c < nsc + nwc; ++c) {
            const uint32_t j = c < nsc ? c * 64u + (uint32_t)lane : lo + (c - nsc) * 64u + (uint32_t)lane;
            bool seen = c < nsc ? j < sink : j < end;
            uint64_t row = 0u;                                       // byte offset of the key's row
            if (seen) {
                const uint32_t page = paged_page(a.c, a.s, s, j >> a.c.page_shift);
                seen = page < a.c.n_pages;
                const uint32_t slot = j & ((1u << a.c.page_shift) - 1u);
                if (seen) row = (uint64_t)page * a.c.page_bytes + (((uint64_t)kvh << a.c.page_shift) + slot) * D * es;
            }
            float x = kNoScore;
            if (seen) {
                float dot = 0.f;
                const uint8_t* const kp = a.c.k + row;
                uint32_t d = 0u;
                for (; d + 16u <= D; d += 16u) {
                    float k[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) k[i] = load_kv_elem(kp, DT, d + (uint32_t)i);
#pragma unroll
                    for (int i = 0; i < 16; ++i) dot = __builtin_fmaf(k[i], q[d + (uint32_t)i], dot);
                }
                for (; d < D; ++d) dot = __builtin_fmaf(load_kv_elem(kp, DT, d), q[d], dot);
                x = a.softcap > 0.f ? a.softcap * tanhf(dot / a.softcap) : dot;
            }
            const float mn = fmaxf(m, wave_max_all(x));
            const float corr = expf(m - mn);
            const float pr = seen ? 0x1p-6f * expf(x - mn) : 0.f;            // (2^23 keys of 2^110 sum to a finite number)
            m = mn;
            l = l * corr + wave_sum_all(pr);
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] *= corr;
            const uint64_t there = __ballot(seen);
            for (int k0 = 0; k0 < 64; k0 += 8) {
                if ((there >> k0 & 0xFFu) == 0u) continue;
                float pk[8];
                uint64_t rk[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {                        // (a key that is not seen: row 0 with its elements left out)
                    pk[k] = __shfl(pr, k0 + k, kWave);
                    rk[k] = (uint64_t)__shfl((unsigned long long)row, k0 + k, kWave);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t d = (uint32_t)lane + 64u * i;
                    if (d >= D) continue;
                    float v[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) v[k] = load_kv_elem(a.c.v + rk[k], DT, d);
#pragma unroll
                    for (int k = 0; k < 8; ++k) acc[i] = __builtin_fmaf(pk[k], there >> (k0 + k) & 1u ? v[k] : 0.f, acc[i]);
                }
            }
        }
    }
    const float inv = l != 0.f ? 1.0f / l : 0.f;                     // (a NaN sum stays one)
    T* const o = reinterpret_cast<T*>(a.o) + (uint64_t)tok * a.o_stride + (uint64_t)head * D;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t d = (uint32_t)lane + 64u * i;
        if (d < D) o[d] = (T)(acc[i] * inv);
    }
}

hipError_t launch_paged_generic(const PagedAttnLaunch& L, hipStream_t stream) {
    if (L.c.head_dim == 0u || L.c.head_dim > 512u || L.n_heads == 0u || L.n_heads % L.c.n_kv_heads != 0u) return hipErrorInvalidValue;
    const uint32_t y = (L.n_heads + 3u) / 4u;
    if (y > 65535u) return hipErrorInvalidValue;
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(L.s.n_tokens, y), dim3(256), 0, stream, L); };
    if (L.c.dtype == kF8) { if (L.io_f16) go(paged_generic_kernel<_Float16, kF8>); else go(paged_generic_kernel<float, kF8>); }
    else if (L.c.dtype == kF16) { if (L.io_f16) go(paged_generic_kernel<_Float16, kF16>); else go(paged_generic_kernel<float, kF16>); }
    else if (L.io_f16) go(paged_generic_kernel<_Float16, kF32>);
    else go(paged_generic_kernel<float, kF32>);
    return hipGetLastError();
}

}  // namespace vfkv
