// Prefill attention over the paged cache: choice of the kernel by cache type, and the join of split rows (paged_prefill.h).
#include "device_utils.h"
#include "paged.h"

namespace vfkv {

// Joins the n_split parts of every row that belongs to a sequence.  head_dim / 4 threads hold four columns each; `per_row` such groups
// share the parts of a row (1: a group per row; more: the whole workgroup on one row, for few rows with many parts).  Eight parts
// are requested at a time.
__global__ __launch_bounds__(256) void paged_rows_merge_kernel(PagedAttnLaunch a, uint32_t n_split, uint32_t per_row) {
    __shared__ float4_t sums[256];
    __shared__ float ls[256], ms[256];
    const uint32_t dr = a.c.head_dim, quads = dr / 4u, groups = 256u / quads, rows_here = groups / per_row;
    const uint32_t grp = threadIdx.x / quads, d = (threadIdx.x % quads) * 4u;
    const uint64_t row = (uint64_t)blockIdx.x * rows_here + grp / per_row;
    const uint32_t first = grp % per_row;
    bool mine = grp < rows_here * per_row && row < (uint64_t)a.s.n_tokens * a.n_heads;
    const uint32_t tok = mine ? (uint32_t)(row / a.n_heads) : 0u, head = mine ? (uint32_t)(row - (uint64_t)tok * a.n_heads) : 0u;
    mine = mine && paged_seq_of(a.s, tok) < a.s.n_seqs;
    float M = kNoScore, L = 0.f;
    float4_t sum = {0.f, 0.f, 0.f, 0.f};
    if (mine) {
        constexpr int AT_ONCE = 8;
        for (uint32_t j0 = first; j0 < n_split; j0 += AT_ONCE * per_row) {
            float m[AT_ONCE], l[AT_ONCE];
            float4_t v[AT_ONCE];
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                const uint32_t j = j0 + (uint32_t)i * per_row;
                const uint64_t at = row * n_split + (j < n_split ? j : j0);
                m[i] = a.scratch_max[at];
                l[i] = a.scratch_sum[at];
                v[i] = *reinterpret_cast<const float4_t*>(a.scratch_out + at * dr + d);
            }
            float mn = M;
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) mn = fmaxf(mn, m[i]);
            const float old = __builtin_amdgcn_exp2f(M - mn);
            M = mn;
            L *= old;
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[i] *= old;
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                if (j0 + (uint32_t)i * per_row >= n_split) break;
                const float f = __builtin_amdgcn_exp2f(m[i] - M);
                L = __builtin_fmaf(l[i], f, L);
#pragma unroll
                for (int k = 0; k < 4; ++k) sum[k] = __builtin_fmaf(v[i][k], f, sum[k]);
            }
        }
    }
    if (per_row > 1u) {
        sums[threadIdx.x] = sum;
        ls[threadIdx.x] = L;
        ms[threadIdx.x] = M;
        __syncthreads();
        if (!mine || first != 0u) return;
        float top = M;
        for (uint32_t x = 1; x < per_row; ++x) top = fmaxf(top, ms[threadIdx.x + x * quads]);
        const float own = __builtin_amdgcn_exp2f(M - top);
        L *= own;
#pragma unroll
        for (int k = 0; k < 4; ++k) sum[k] *= own;
        for (uint32_t x = 1; x < per_row; ++x) {
            const float f = __builtin_amdgcn_exp2f(ms[threadIdx.x + x * quads] - top);
            const float4_t v = sums[threadIdx.x + x * quads];
            L = __builtin_fmaf(ls[threadIdx.x + x * quads], f, L);
#pragma unroll
            for (int k = 0; k < 4; ++k) sum[k] = __builtin_fmaf(v[k], f, sum[k]);
        }
    }
    if (!mine) return;
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
    const uint32_t groups = 256u / (L.c.head_dim / 4u);
    const uint64_t rows = (uint64_t)L.s.n_tokens * L.n_heads;
    // a group takes eight parts per trip to memory: a whole workgroup per row where that is not enough and the rows are too few to
    // fill the card (7 tokens over 4 000 keys in 31 parts: 26.2 -> 16.9 us; 512 tokens in nine parts: 28.7 against 48.6 us)
    const uint32_t per_row = n_split > 8u && rows < 256u * groups ? groups : 1u;
    const uint32_t here = groups / per_row;
    hipLaunchKernelGGL(paged_rows_merge_kernel, dim3((uint32_t)((rows + here - 1u) / here)), dim3(256), 0, stream, L, n_split, per_row);
    return hipGetLastError();
}

hipError_t launch_paged_prefill(const PagedAttnLaunch& L, hipStream_t stream) {
    if ((uint64_t)L.s.n_tokens * L.n_heads > 1u << 30) return hipErrorInvalidValue;
    if (L.c.dtype == kF8) return launch_paged_prefill_byte(L, stream);
    return L.c.dtype == kF16 ? launch_paged_prefill_half(L, stream) : launch_paged_prefill_full(L, stream);
}

}  // namespace vfkv
