// Attention over the paged cache: the generic form.  (paged_decode.hip and paged_prefill.h hold the matrix-core kernels.)
#include "device_utils.h"
#include "paged.h"

namespace vfkv {

// ---- generic form --------------------------------------------------------------------------------
// One wavefront per (token, head), for the head widths and alignments the matrix-core kernels do not take.  64 keys at a time: a
// lane forms the whole score of one key, then the lanes share the value columns; running maximum and sum in f32.
template <typename T>
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
    const uint32_t es = elem_size(a.c.dtype);
    float* const q = q_lds[w];
    for (uint32_t d = lane; d < D; d += kWave)
        q[d] = (float)reinterpret_cast<const T*>(a.q)[(uint64_t)tok * a.q_stride + (uint64_t)head * D + d] * a.scale;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    float m = kMasked, l = 0.f;
    if (pos >= 0) {
        const uint32_t p = (uint32_t)pos, lo = paged_window_lo(a.window, p);
        const uint32_t sink = a.n_sink < lo ? a.n_sink : lo;
        // chunks of the first tokens, then chunks of the window
        const uint32_t nsc = (sink + 63u) / 64u, nwc = (p + 1u - lo + 63u) / 64u;
        for (uint32_t c = 0; c < nsc + nwc; ++c) {
            const uint32_t j = c < nsc ? c * 64u + (uint32_t)lane : lo + (c - nsc) * 64u + (uint32_t)lane;
            bool seen = c < nsc ? j < sink : j <= p;
            uint64_t row = 0u;                                       // byte offset of the key's row
            if (seen) {
                const uint32_t page = paged_page(a.c, a.s, s, j >> a.c.page_shift);
                seen = page < a.c.n_pages;
                const uint32_t slot = j & ((1u << a.c.page_shift) - 1u);
                if (seen) row = (uint64_t)page * a.c.page_bytes + (((uint64_t)kvh << a.c.page_shift) + slot) * D * es;
            }
            float x = kMasked;
            if (seen) {
                float dot = 0.f;
                for (uint32_t d = 0; d < D; ++d) dot = __builtin_fmaf(load_kv_elem(a.c.k + row, a.c.dtype, d), q[d], dot);
                x = a.softcap > 0.f ? a.softcap * tanhf(dot / a.softcap) : dot;
            }
            const float mn = fmaxf(m, wave_max_all(x));
            const float corr = expf(m - mn);
            const float pr = seen ? expf(x - mn) : 0.f;
            m = mn;
            l = l * corr + wave_sum_all(pr);
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] *= corr;
            uint64_t todo = __ballot(seen);
            while (todo != 0u) {
                const int k = __builtin_ctzll(todo);
                todo &= todo - 1u;
                const float pk = __shfl(pr, k, kWave);
                const uint64_t rk = (uint64_t)__shfl((unsigned long long)row, k, kWave);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t d = (uint32_t)lane + 64u * i;
                    if (d < D) acc[i] = __builtin_fmaf(pk, load_kv_elem(a.c.v + rk, a.c.dtype, d), acc[i]);
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
    if (L.io_f16) hipLaunchKernelGGL(paged_generic_kernel<_Float16>, dim3(L.s.n_tokens, y), dim3(256), 0, stream, L);
    else hipLaunchKernelGGL(paged_generic_kernel<float>, dim3(L.s.n_tokens, y), dim3(256), 0, stream, L);
    return hipGetLastError();
}

}  // namespace vfkv
