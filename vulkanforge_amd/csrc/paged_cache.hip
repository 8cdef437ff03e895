// Kernels that fill and move pages of the paged cache: page copies, and norm + rotation + append of a batch of tokens.
#include <type_traits>

#include "device_utils.h"
#include "paged.h"

namespace vfkv {

// ---- page copies -------------------------------------------------------------------------------
// dst page <- src page for all layers, K and V: pure traffic, one read and one write per byte.  The pairs travel as kernel
// arguments: no upload, and a captured call keeps its own list.  blockIdx.y = pair, blockIdx.z = layer and tensor, blockIdx.x =
// share of the page.  A page of one layer is contiguous; with fewer rows it is n_kv_heads pieces, each at a multiple of
// page_size rows, hence 16-byte aligned whatever the row length.  Measured: 200 pages of 128 KiB in 32 layers (3.36 GB read and written)
// 632 us = 5.3 TB/s, what a copy of 1 GiB reaches (5.2); four partial pages (fork) 3.8 us.
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
constexpr int kWriteWaves = 4;

// cos and sin of pair p of a token, scaled.
__device__ __forceinline__ void pair_angle(const PagedWriteLaunch& a, uint32_t p, uint32_t tok, int64_t pos, float& cs, float& sn) {
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
    sincospif((float)(2.0 * (turns - rint(turns))), &sn, &cs);
    cs *= a.attn_factor;
    sn *= a.attn_factor;
}

// Four elements of a row in the cache type.
__device__ __forceinline__ void store_quad(uint8_t* dst, uint32_t dtype, uint32_t e, const float4_t& x) {
    if (dtype == kF8) *reinterpret_cast<uint32_t*>(dst + e) = pack4_e4m3(x[0], x[1], x[2], x[3]);
    else if (dtype == kF16) *reinterpret_cast<u32x2*>(dst + 2u * e) = u32x2{f32_to_h16_bits(x[0]) | f32_to_h16_bits(x[1]) << 16,
                                                                        f32_to_h16_bits(x[2]) | f32_to_h16_bits(x[3]) << 16};
    else *reinterpret_cast<float4_t*>(dst + 4u * e) = x;
}
template <typename T>
__device__ __forceinline__ float4_t load_quad(const void* p, uint64_t i) {
    if constexpr (sizeof(T) == 4) return *reinterpret_cast<const float4_t*>(reinterpret_cast<const float*>(p) + i);
    const half4_t h = *reinterpret_cast<const half4_t*>(reinterpret_cast<const _Float16*>(p) + i);
    return float4_t{(float)h[0], (float)h[1], (float)h[2], (float)h[3]};
}

// Rows in quads: LPR lanes per row, two quads of four elements per lane, 64 / LPR rows per wavefront at a time.  A lane of the
// rotated part holds both elements of its four pairs (quads p and p + rotary_dim / 2 apart, or eight neighbours), so nothing
// crosses lanes but the sum of squares; the pairs' cos and sin are computed once per token and wavefront, one per lane, and passed
// round.  A wavefront takes every `parts`-th group of rows of its token and requests kAhead of them before it works on the first.
// Measured: 5 692 tokens, 32 / 8 / 128, f16 rows into F16 pages 36.5 us = 3.8 TB/s (element by element: 142 us; two or four steps
// ahead and two to three wavefronts per token measured the same or slower: the vector units are busy half the time, a token's chain of
// steps the other half); 32 decode tokens 5.8 us.
constexpr int kAhead = 3;
template <typename T, int LPR>
__global__ __launch_bounds__(kWriteWaves * kWave) void paged_write_quads_kernel(PagedWriteLaunch a, uint32_t parts) {
    constexpr uint32_t RPI = 64 / LPR;                          // rows per step
    const int lane = threadIdx.x & 63;
    const uint32_t unit = blockIdx.x * kWriteWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t tok = unit / parts, part = unit - tok * parts;
    if (tok >= a.s.n_tokens) return;
    const uint32_t c = (uint32_t)lane % LPR, sub = (uint32_t)lane / LPR;
    const uint32_t D = a.c.head_dim, half = a.rotary_dim / 2u, quads = half / 4u;
    const bool on = c < D / 8u, turn = c < quads;
    const uint32_t e0 = !on ? 0u : turn ? (a.mode == 2u ? 4u * c : 8u * c) : a.rotary_dim + 8u * (c - quads);
    const uint32_t e1 = !on ? 0u : turn && a.mode == 2u ? half + 4u * c : e0 + 4u;
    // steps: RPI query rows each, then key rows, then value rows
    const uint32_t nq = a.q ? a.n_heads : 0u, hkv = a.c.n_kv_heads;
    const uint32_t q_steps = (nq + RPI - 1u) / RPI, k_steps = (hkv + RPI - 1u) / RPI, steps = q_steps + 2u * k_steps;

    float4_t x0[kAhead], x1[kAhead];
    auto load = [&](int i, uint32_t st) {                       // (steps past the last read the last again)
        st = st < steps ? st : steps - 1u;
        const bool is_q = st < q_steps, is_v = st >= q_steps + k_steps;
        const uint32_t r = (is_q ? st : is_v ? st - q_steps - k_steps : st - q_steps) * RPI + sub, n = is_q ? nq : hkv;
        const T* const src = reinterpret_cast<const T*>(is_q ? a.q : is_v ? a.v : a.k) + (uint64_t)tok * (is_q ? a.q_stride : is_v ? a.v_stride : a.k_stride);
        const uint32_t at = (r < n ? r : n - 1u) * D;
        x0[i] = load_quad<T>(src, at + e0);
        x1[i] = load_quad<T>(src, at + e1);
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) load(i, part + (uint32_t)i * parts);

    // ---- the token's sequence: 64 offsets at a time
    uint32_t s = tok;
    if (a.s.q_offsets != nullptr) {
        s = 0u;
        for (uint32_t base = 0; base < a.s.n_seqs; base += 64u) {
            const uint32_t i = base + (uint32_t)lane;
            s += (uint32_t)__builtin_popcountll(__ballot(i < a.s.n_seqs && a.s.q_offsets[i + 1u] <= (int32_t)tok));
        }
    }
    s = __builtin_amdgcn_readfirstlane(s);
    if (s >= a.s.n_seqs) return;                                // a padding row: left as it was
    uint32_t r0, r1;
    paged_rows(a.s, s, r0, r1);
    if (tok < r0 || tok >= r1) return;
    const int64_t pos = (int64_t)paged_kv_len(a.s, s) - (int64_t)(r1 - tok);
    const uint32_t page = pos >= 0 && pos < (int64_t)a.s.limit ? paged_page(a.c, a.s, s, (uint32_t)pos >> a.c.page_shift) : a.c.n_pages;
    const uint32_t slot = (uint32_t)pos & ((1u << a.c.page_shift) - 1u);
    const uint64_t page_at = (uint64_t)(page < a.c.n_pages ? page : 0u) * a.c.page_bytes;
    const uint32_t row_b = D * elem_size(a.c.dtype);

    // ---- angles: lane (c, sub) computes pair 4 c + sub (+ RPI, ...), then every lane collects its four
    float cs[4], sn[4];
    {
        constexpr int MINE = RPI >= 4u ? 1 : 4 / (int)RPI;
        float mc[MINE], ms[MINE];
#pragma unroll
        for (int i = 0; i < MINE; ++i) {
            const uint32_t j = sub % 4u + (uint32_t)i * RPI;
            mc[i] = 1.f;
            ms[i] = 0.f;
            if (turn && j < 4u) pair_angle(a, 4u * c + j, tok, pos, mc[i], ms[i]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int from = (int)((uint32_t)j % (RPI < 4u ? RPI : 4u) * LPR + c);
            cs[j] = __shfl(mc[RPI >= 4u ? 0 : j / (int)RPI], from, kWave);
            sn[j] = __shfl(ms[RPI >= 4u ? 0 : j / (int)RPI], from, kWave);
        }
    }
    const float4_t one = {1.f, 1.f, 1.f, 1.f};
    const float4_t wq0 = a.q_weight && on ? load_quad<float>(a.q_weight, e0) : one, wq1 = a.q_weight && on ? load_quad<float>(a.q_weight, e1) : one;
    const float4_t wk0 = a.k_weight && on ? load_quad<float>(a.k_weight, e0) : one, wk1 = a.k_weight && on ? load_quad<float>(a.k_weight, e1) : one;

    auto row = [&](auto kind, int i, uint32_t r) {
        constexpr int KIND = decltype(kind)::value;             // 0: query, 1: key, 2: value
        float4_t y0 = x0[i], y1 = x1[i];
        if (KIND != 2 && (KIND == 0 ? a.q_weight : a.k_weight) != nullptr) {
            float ss = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) ss = __builtin_fmaf(y0[j], y0[j], __builtin_fmaf(y1[j], y1[j], ss));
            ss = group_sum<LPR>(on ? ss : 0.f);
            const float f = 1.0f / sqrtf(ss / (float)D + a.eps);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                y0[j] = (f * y0[j]) * (KIND == 0 ? wq0[j] : wk0[j]);
                y1[j] = (f * y1[j]) * (KIND == 0 ? wq1[j] : wk1[j]);
            }
        }
        if (KIND != 2 && turn) {
            if (a.mode == 2u) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float p = y0[j], q = y1[j];
                    y0[j] = __builtin_fmaf(p, cs[j], -(q * sn[j]));
                    y1[j] = __builtin_fmaf(p, sn[j], q * cs[j]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float4_t& y = j < 2 ? y0 : y1;
                    const int k = 2 * (j % 2);
                    const float p = y[k], q = y[k + 1];
                    y[k] = __builtin_fmaf(p, cs[j], -(q * sn[j]));
                    y[k + 1] = __builtin_fmaf(p, sn[j], q * cs[j]);
                }
            }
        }
        if (!on || r >= (KIND == 0 ? nq : hkv)) return;
        if constexpr (KIND == 0) {
            T* const out = reinterpret_cast<T*>(a.q_out) + (uint64_t)tok * a.q_out_stride;
            if constexpr (sizeof(T) == 4) {
                *reinterpret_cast<float4_t*>(out + (r * D + e0)) = y0;
                *reinterpret_cast<float4_t*>(out + (r * D + e1)) = y1;
            } else {
                *reinterpret_cast<half4_t*>(out + (r * D + e0)) = half4_t{(_Float16)y0[0], (_Float16)y0[1], (_Float16)y0[2], (_Float16)y0[3]};
                *reinterpret_cast<half4_t*>(out + (r * D + e1)) = half4_t{(_Float16)y1[0], (_Float16)y1[1], (_Float16)y1[2], (_Float16)y1[3]};
            }
        } else if (page < a.c.n_pages) {
            uint8_t* const dst = const_cast<uint8_t*>(KIND == 2 ? a.c.v : a.c.k) + page_at + (((uint64_t)r << a.c.page_shift) + slot) * row_b;
            store_quad(dst, a.c.dtype, e0, y0);
            store_quad(dst, a.c.dtype, e1, y1);
        }
    };
    for (uint32_t st = part; st < steps; st += kAhead * parts) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const uint32_t u = st + (uint32_t)i * parts;
            if (u < q_steps) row(std::integral_constant<int, 0>{}, i, u * RPI + sub);
            else if (u < q_steps + k_steps) row(std::integral_constant<int, 1>{}, i, (u - q_steps) * RPI + sub);
            else if (u < steps) row(std::integral_constant<int, 2>{}, i, (u - q_steps - k_steps) * RPI + sub);
            load(i, u + (uint32_t)kAhead * parts);
        }
    }
}

// Rows of any width and alignment, element by element through LDS.

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
        for (uint32_t p = tid; p < half; p += kWriteWaves * kWave) pair_angle(a, p, tok, pos, cs_lds[p], sn_lds[p]);
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
    if (pos < 0 || pos >= (int64_t)a.s.limit) return;
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
    const uint32_t D = L.c.head_dim;
    const uintptr_t mask = L.io_f16 ? 7u : 15u;                 // one quad
    const uintptr_t all = (uintptr_t)L.q | (uintptr_t)L.q_out | (uintptr_t)L.k | (uintptr_t)L.v;
    const uintptr_t weights = (uintptr_t)L.q_weight | (uintptr_t)L.k_weight;
    if (D % 8u == 0u && L.rotary_dim % 8u == 0u && (all & mask) == 0u && (weights & 15u) == 0u &&
        ((L.q_stride | L.q_out_stride | L.k_stride | L.v_stride) & 3u) == 0u) {
        const uint32_t lpr = D <= 64u ? 8u : D <= 128u ? 16u : D <= 256u ? 32u : 64u, rpi = 64u / lpr;
        // few tokens: a token's rows go to several wavefronts (four wavefronts per SIMD fill the card)
        const uint32_t steps = ((L.q ? L.n_heads : 0u) + rpi - 1u) / rpi + 2u * ((L.c.n_kv_heads + rpi - 1u) / rpi);
        uint32_t parts = (4096u + L.s.n_tokens - 1u) / L.s.n_tokens;
        if (parts > steps) parts = steps;
        const uint64_t blocks = ((uint64_t)L.s.n_tokens * parts + kWriteWaves - 1u) / kWriteWaves;
        if (blocks <= 0x7FFFFFFFu && (uint64_t)L.s.n_tokens * parts <= 0xFFFFFFFFu) {
            auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((uint32_t)blocks), dim3(kWriteWaves * kWave), 0, stream, L, parts); };
            if (L.io_f16) {
                if (lpr == 8u) go(paged_write_quads_kernel<_Float16, 8>);
                else if (lpr == 16u) go(paged_write_quads_kernel<_Float16, 16>);
                else if (lpr == 32u) go(paged_write_quads_kernel<_Float16, 32>);
                else go(paged_write_quads_kernel<_Float16, 64>);
            } else {
                if (lpr == 8u) go(paged_write_quads_kernel<float, 8>);
                else if (lpr == 16u) go(paged_write_quads_kernel<float, 16>);
                else if (lpr == 32u) go(paged_write_quads_kernel<float, 32>);
                else go(paged_write_quads_kernel<float, 64>);
            }
            return hipGetLastError();
        }
    }
    const uint32_t y = (units + kWriteWaves - 1u) / kWriteWaves;
    if (y > 65535u) return hipErrorInvalidValue;
    if (L.io_f16) hipLaunchKernelGGL(paged_write_kernel<_Float16>, dim3(L.s.n_tokens, y), dim3(kWriteWaves * kWave), 0, stream, L);
    else hipLaunchKernelGGL(paged_write_kernel<float>, dim3(L.s.n_tokens, y), dim3(kWriteWaves * kWave), 0, stream, L);
    return hipGetLastError();
}

}  // namespace vfkv
