// Kernels that fill and move pages of the paged cache: page copies, and norm + rotation + append of a batch of tokens.
#include "device_utils.h"
#include "paged.h"

namespace vfkv {

// ---- page copies -------------------------------------------------------------------------------
// dst page <- src page for all layers, K and V: pure traffic, one read and one write per byte.  The pairs travel as kernel
// arguments: no upload, and a captured call keeps its own list.  blockIdx.y = pair, blockIdx.z = layer and tensor, blockIdx.x =
// share of the page.  A page of one layer is contiguous; with fewer rows it is n_kv_heads pieces, each at a multiple of
// page_size rows, hence 16-byte aligned whatever the row length.
struct CopyArgs {
    uint8_t* buf[2];
    uint64_t layer_bytes, page_bytes;
    uint32_t page_size, row_bytes, n_kv_heads;
    uint32_t src[kCopyPairs], dst[kCopyPairs];
    uint16_t rows[kCopyPairs];
};
constexpr uint32_t kCopyShare = 16384u;    // bytes per workgroup: four 16-byte loads in flight per thread

__global__ __launch_bounds__(256) void paged_copy_kernel(CopyArgs a) {
    const uint32_t i = blockIdx.y;
    uint8_t* const base = a.buf[blockIdx.z & 1u] + (uint64_t)(blockIdx.z >> 1) * a.layer_bytes;
    const uint8_t* const src = base + (uint64_t)a.src[i] * a.page_bytes;
    uint8_t* const dst = base + (uint64_t)a.dst[i] * a.page_bytes;
    const uint32_t rows = a.rows[i];
    const bool whole = rows == a.page_size;
    const uint64_t piece = whole ? a.page_bytes : (uint64_t)rows * a.row_bytes;
    const uint64_t stride = (uint64_t)a.page_size * a.row_bytes;
    const uint32_t pieces = whole ? 1u : a.n_kv_heads;
    const uint64_t vecs = (piece + 15u) / 16u;               // the last one of a piece may be ragged
    const uint64_t total = vecs * pieces;
    const uint64_t step = (uint64_t)gridDim.x * 1024u;
    for (uint64_t b = (uint64_t)blockIdx.x * 1024u; b < total; b += step) {
        u32x4 x[4];
        uint64_t off[4];
        uint32_t len[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint64_t e = b + (uint64_t)j * 256u + threadIdx.x;
            len[j] = 0u;
            if (e < total) {
                const uint64_t p = whole ? 0u : e / vecs, in = (e - p * vecs) * 16u;
                off[j] = p * stride + in;
                len[j] = piece - in < 16u ? (uint32_t)(piece - in) : 16u;
                if (len[j] == 16u) x[j] = *reinterpret_cast<const u32x4*>(src + off[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (len[j] == 16u) *reinterpret_cast<u32x4*>(dst + off[j]) = x[j];
            else for (uint32_t t = 0; t < len[j]; ++t) dst[off[j] + t] = src[off[j] + t];
        }
    }
}

hipError_t launch_paged_copy(const PagedCopyLaunch& L, hipStream_t stream) {
    if (L.n == 0u) return hipSuccess;
    if (L.n > kCopyPairs || L.n_layers > 32767u) return hipErrorInvalidValue;
    CopyArgs a;
    a.buf[0] = L.k; a.buf[1] = L.v;
    a.layer_bytes = L.layer_bytes; a.page_bytes = L.page_bytes;
    a.page_size = L.page_size; a.row_bytes = L.row_bytes; a.n_kv_heads = L.n_kv_heads;
    uint32_t most = 0u;
    for (uint32_t i = 0; i < L.n; ++i) {
        a.src[i] = L.src[i]; a.dst[i] = L.dst[i];
        const uint32_t r = L.rows ? L.rows[i] : L.page_size;
        a.rows[i] = (uint16_t)r;
        most = r > most ? r : most;
    }
    if (most == 0u) return hipSuccess;
    const uint64_t bytes = (uint64_t)most * L.row_bytes * L.n_kv_heads;
    uint64_t x = (bytes + kCopyShare - 1u) / kCopyShare;
    if (x > 65535u) x = 65535u;
    hipLaunchKernelGGL(paged_copy_kernel, dim3((uint32_t)x, L.n, 2u * L.n_layers), dim3(256), 0, stream, a);
    return hipGetLastError();
}

// ---- norm + rotation + append --------------------------------------------------------------------
// One wavefront per (token, tensor, head) row, four rows of a token per workgroup, as rope_append_kernel does for the contiguous
// cache.  Bound by its traffic: every element is read once and written once.
//
// Angle of pair p: pos[axis] * 2^(p * log2_step), in turns and in 64 bits up to the fraction of a turn, because an f32 angle of
// 10^5 radians is off by up to 4e-3; the fraction is then exact to 2^-25 of a turn in f32.
struct WriteArgs {
    PagedWriteLaunch L;
};
constexpr int kWriteWaves = 4;

template <typename T>
__device__ __forceinline__ float io_load(const void* p, uint64_t i) { return (float)reinterpret_cast<const T*>(p)[i]; }

template <typename T>
__global__ __launch_bounds__(kWriteWaves * kWave) void paged_write_kernel(PagedWriteLaunch a) {
    __shared__ float cs_lds[256], sn_lds[256];
    __shared__ float rows[kWriteWaves][512];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const uint32_t tok = blockIdx.x;
    const uint32_t s = paged_seq_of(a.s, tok);
    if (s >= a.s.n_seqs) return;                                  // a padding row: left as it was
    uint32_t r0, r1;
    paged_rows(a.s, s, r0, r1);
    const int64_t pos = (int64_t)paged_kv_len(a.s, s) - (int64_t)(r1 - tok);
    const uint32_t D = a.c.head_dim, half = a.rotary_dim / 2u;
    const uint32_t nq = a.q ? a.n_heads : 0u, hkv = a.c.n_kv_heads;
    if (blockIdx.y * kWriteWaves < nq + hkv) {
        for (uint32_t p = tid; p < half; p += kWriteWaves * kWave) {
            uint32_t axis = 0u;
            if (a.n_axes > 1u) {
                if (a.interleaved) {
                    const uint32_t x = p % a.n_axes;
                    axis = p / a.n_axes < a.section[x] ? x : 0u;
                } else {
                    uint32_t end = a.section[0];
                    while (axis + 1u < a.n_axes && p >= end) end += a.section[++axis];
                }
            }
            const double at = a.positions ? (double)a.positions[(uint64_t)axis * a.s.n_tokens + tok] : (double)pos;
            double turns = at * exp2((double)p * a.log2_step) * 0.15915494309189535 * (double)a.freq_scale;
            if (a.freq_factors) turns /= (double)a.freq_factors[p];
            const float t = (float)(2.0 * (turns - rint(turns)));
            float sn, cs;
            sincospif(t, &sn, &cs);
            cs_lds[p] = cs * a.attn_factor;
            sn_lds[p] = sn * a.attn_factor;
        }
    }
    __syncthreads();
    const uint32_t u = blockIdx.y * kWriteWaves + w;
    if (u >= nq + 2u * hkv) return;
    const bool is_q = u < nq, is_v = u >= nq + hkv;
    const uint32_t head = is_q ? u : is_v ? u - nq - hkv : u - nq;
    const void* const src = is_q ? a.q : is_v ? a.v : a.k;
    const uint64_t off = (uint64_t)tok * (is_q ? a.q_stride : is_v ? a.v_stride : a.k_stride) + (uint64_t)head * D;
    const float* const weight = is_q ? a.q_weight : is_v ? nullptr : a.k_weight;
    float* const row = rows[w];
    float ss = 0.f;
    for (uint32_t d = lane; d < D; d += kWave) {
        const float x = io_load<T>(src, off + d);
        row[d] = x;
        ss = __builtin_fmaf(x, x, ss);
    }
    if (weight != nullptr) {
        ss = wave_sum_all(ss);
        const float r = 1.0f / sqrtf(ss / (float)D + a.eps);
        for (uint32_t d = lane; d < D; d += kWave) row[d] = (r * row[d]) * weight[d];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (!is_v) {
        for (uint32_t p = lane; p < half; p += kWave) {
            const uint32_t i0 = a.mode == 2u ? p : 2u * p, i1 = a.mode == 2u ? p + half : 2u * p + 1u;
            const float x0 = row[i0], x1 = row[i1], cs = cs_lds[p], sn = sn_lds[p];
            row[i0] = __builtin_fmaf(x0, cs, -(x1 * sn));
            row[i1] = __builtin_fmaf(x0, sn, x1 * cs);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    if (is_q) {
        T* const out = reinterpret_cast<T*>(a.q_out) + (uint64_t)tok * a.q_out_stride + (uint64_t)head * D;
        for (uint32_t d = lane; d < D; d += kWave) out[d] = (T)row[d];
        return;
    }
    if (pos < 0) return;
    const uint32_t page = paged_page(a.c, a.s, s, (uint32_t)pos >> a.c.page_shift);
    if (page >= a.c.n_pages) return;
    const uint32_t slot = (uint32_t)pos & ((1u << a.c.page_shift) - 1u);
    const uint32_t es = elem_size(a.c.dtype);
    uint8_t* const dst = const_cast<uint8_t*>(is_v ? a.c.v : a.c.k) + (uint64_t)page * a.c.page_bytes +
                         (((uint64_t)head << a.c.page_shift) + slot) * D * es;
    for (uint32_t d = lane; d < D; d += kWave) {
        if (a.c.dtype == kF8) dst[d] = (uint8_t)pack4_e4m3(row[d], 0.f, 0.f, 0.f);
        else if (a.c.dtype == kF16) reinterpret_cast<uint16_t*>(dst)[d] = (uint16_t)f32_to_h16_bits(row[d]);
        else reinterpret_cast<float*>(dst)[d] = row[d];
    }
}

hipError_t launch_paged_write(const PagedWriteLaunch& L, hipStream_t stream) {
    if (L.s.n_tokens == 0u) return hipSuccess;
    if (L.c.head_dim == 0u || L.c.head_dim > 512u || L.rotary_dim > L.c.head_dim || L.rotary_dim % 2u != 0u) return hipErrorInvalidValue;
    const uint32_t units = (L.q ? L.n_heads : 0u) + 2u * L.c.n_kv_heads;
    const uint32_t y = (units + kWriteWaves - 1u) / kWriteWaves;
    if (y > 65535u) return hipErrorInvalidValue;
    if (L.io_f16) hipLaunchKernelGGL(paged_write_kernel<_Float16>, dim3(L.s.n_tokens, y), dim3(kWriteWaves * kWave), 0, stream, L);
    else hipLaunchKernelGGL(paged_write_kernel<float>, dim3(L.s.n_tokens, y), dim3(kWriteWaves * kWave), 0, stream, L);
    return hipGetLastError();
}

}  // namespace vfkv
