// Prefill attention over the paged cache: choice of the kernel by cache type, and the join of split rows (paged_prefill.h).
#include "device_utils.h"
#include "paged.h"

namespace vfkv {

// Joins the n_split parts of every row that belongs to a sequence: head_dim / 4 threads per row.
__global__ __launch_bounds__(256) void paged_rows_merge_kernel(PagedAttnLaunch a, uint32_t n_split) {
    const uint32_t dr = a.c.head_dim, quads = dr / 4u, per = 256u / quads;
    const uint32_t grp = threadIdx.x / quads, d = (threadIdx.x % quads) * 4u;
    const uint64_t row = (uint64_t)blockIdx.x * per + grp;
    if (grp >= per || row >= (uint64_t)a.s.n_tokens * a.n_heads) return;
    const uint32_t tok = (uint32_t)(row / a.n_heads), head = (uint32_t)(row - (uint64_t)tok * a.n_heads);
    if (paged_seq_of(a.s, tok) >= a.s.n_seqs) return;
    const float* const ms = a.scratch_max + row * n_split;
    const float* const ls = a.scratch_sum + row * n_split;
    float M = ms[0];
    for (uint32_t j = 1; j < n_split; ++j) M = fmaxf(M, ms[j]);
    float L = 0.f;
    float4_t sum = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t j = 0; j < n_split; ++j) {
        const float f = __builtin_amdgcn_exp2f(ms[j] - M);
        const float4_t v = *reinterpret_cast<const float4_t*>(a.scratch_out + (row * n_split + j) * dr + d);
        L = __builtin_fmaf(ls[j], f, L);
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] = __builtin_fmaf(v[i], f, sum[i]);
    }
    const float inv = L != 0.f ? 1.0f / L : 0.f;
    const uint64_t at = (uint64_t)tok * a.o_stride + (uint64_t)head * dr + d;
    if (a.io_f16) {
        half4_t h;
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = (_Float16)(sum[i] * inv);
        *reinterpret_cast<half4_t*>(reinterpret_cast<_Float16*>(a.o) + at) = h;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] *= inv;
        *reinterpret_cast<float4_t*>(reinterpret_cast<float*>(a.o) + at) = sum;
    }
}

hipError_t launch_paged_rows_merge(const PagedAttnLaunch& L, uint32_t n_split, hipStream_t stream) {
    const uint32_t per = 256u / (L.c.head_dim / 4u);
    const uint64_t rows = (uint64_t)L.s.n_tokens * L.n_heads;
    hipLaunchKernelGGL(paged_rows_merge_kernel, dim3((uint32_t)((rows + per - 1u) / per)), dim3(256), 0, stream, L, n_split);
    return hipGetLastError();
}

hipError_t launch_paged_prefill(const PagedAttnLaunch& L, hipStream_t stream) {
    if ((uint64_t)L.s.n_tokens * L.n_heads > 0xFFFFFFFFull) return hipErrorInvalidValue;
    if (L.c.dtype == kF8) return launch_paged_prefill_byte(L, stream);
    return L.c.dtype == kF16 ? launch_paged_prefill_half(L, stream) : launch_paged_prefill_full(L, stream);
}

}  // namespace vfkv
