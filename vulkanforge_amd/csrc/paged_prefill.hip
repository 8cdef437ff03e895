// Prefill attention over the paged cache: a ragged batch of chunks, causal, with a window per query and first tokens kept.
//
// o[r] = sum_j softmax_j(scale q[r].k_j) v_j over the keys row r sees; 4 * head_dim flop per visible (query row, key) pair, so
// for chunks of any length the matrix cores bound it.
//
//   - The query heads of one KV head and the tokens of a chunk form one line of rows (token major): a workgroup takes a block of
//     R = 128 NQ consecutive rows of one sequence and one KV head, a wavefront 32 NQ of them.  K and V are shared by the whole
//     group, and short chunks (drafted tokens) fill the tiles with heads.  Blocks are numbered by a prefix sum over the
//     batch that every workgroup forms itself (the offsets are device data), the last block of a sequence first: it has the most keys.
//   - Keys pass through LDS in tiles of KT, as f16 (or f32), once for all rows of the workgroup: global loads of tile t + 1 run
//     during the products of tile t, two LDS buffers, one barrier per tile.  A 16-key tile lies in one page, whose number is a
//     scalar load two tiles ahead.
//   - S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_32x32x16_f16: the scores of a row stay in one lane and its opposite half, P is
//     already where the second product wants it, V^T comes from the transposing LDS read.
//   - f16 queries enter as they are and the weights as f16 (half a step of 2^-11 per weight, like the output's own rounding).  f32
//     queries enter as f16 value + remainder, and so do the weights: f32-level accuracy for twice the products.
//     F32 caches use the f32 matrix instruction.
//   - The running maximum is only raised when a score exceeds it by 2^8; weights are kept times 2^6 (see paged_decode.hip).
//   - Few rows over many keys: the tiles are cut into n_split parts over more workgroups and joined by paged_rows_merge_kernel.
#include "device_utils.h"
#include "paged.h"

namespace vfkv {

namespace {

constexpr float kRaise = 8.f, kBias = 6.f;  // log2

template <int DT, int D, int KT>
struct PreShape {
    static constexpr int ES = DT == kF32 ? 4 : DT == kF16 ? 2 : 1;
    static constexpr int LE = DT == kF32 ? 4 : 2;              // bytes per element in LDS
    static constexpr int CPR = D * ES / 16;                    // 16-byte chunks per cache row
    static constexpr int RPP = 256 / CPR;                      // rows per staging pass
    static constexpr int NP = KT / RPP;                        // passes per tile and tensor
    // pitches: 16-byte reads of eight K rows, and reads of four (f16) / two (f32, four rows apart) V rows, hit distinct banks
    static constexpr int KPITCH = D * LE + 16;                 // bytes
    static constexpr int VPITCH = D * LE + (DT == kF32 ? 32 : 64);
    static constexpr int BUF = KT * (KPITCH + VPITCH);         // one buffer: K tile, V tile
    static_assert(KT % RPP == 0 || RPP > KT, "whole passes");
};

__device__ __forceinline__ float max_over_halves(float x) {
    float y = x;
    swap32(x, y);
    return fmaxf(x, y);
}

}  // namespace

// Exclusive prefix sums of the row blocks of the sequences, by the whole workgroup.
__device__ __forceinline__ void block_prefix(const PagedAttnLaunch& a, uint32_t group, uint32_t rows, uint32_t* pre, uint32_t* wave_sum, int tid) {
    const int lane = tid & 63, w = tid >> 6;
    uint32_t carry = 0u;
    for (uint32_t base = 0; base < a.s.n_seqs; base += 256u) {
        const uint32_t s = base + (uint32_t)tid;
        uint32_t x = 0u;
        if (s < a.s.n_seqs) {
            uint32_t lo, hi;
            paged_rows(a.s, s, lo, hi);
            x = (uint32_t)(((uint64_t)(hi - lo) * group + rows - 1u) / rows);
        }
        const uint32_t mine = x;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const uint32_t y = __shfl_up(x, off, kWave);
            if (lane >= off) x += y;
        }
        if (lane == 63) wave_sum[w] = x;
        __syncthreads();
        uint32_t before = carry;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i < w) before += wave_sum[i];
            carry += wave_sum[i];
        }
        if (s < a.s.n_seqs) pre[s] = before + x - mine;
        __syncthreads();
    }
    if (tid == 0) pre[a.s.n_seqs] = carry;
    __syncthreads();
}

template <int DT, int D, bool IOF16, int NQ, int KT, int MINW>
__global__ __launch_bounds__(256, MINW) void paged_prefill_kernel(PagedAttnLaunch a, uint32_t n_split) {
    using Z = PreShape<DT, D, KT>;
    constexpr bool F32C = DT == kF32;
    constexpr bool PAIR = !IOF16 && !F32C;                   // queries and weights as value + remainder
    constexpr int NB = KT / 32;                              // 32-key blocks per tile
    constexpr int DT32 = D / 32;
    constexpr uint32_t R = 128u * NQ;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];   // two buffers, then the prefix sums
    __shared__ uint32_t wave_sum[4];
    __shared__ uint32_t odd_tile[2];                         // tile number + 1 when the buffer's V holds an infinity or NaN
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n32 = lane & 31, hf = lane >> 5;
    const uint32_t group = a.n_heads / a.c.n_kv_heads, kvh = blockIdx.x;
    const uint32_t dr = a.c.head_dim;
    uint32_t* const pre = reinterpret_cast<uint32_t*>(lds + 2 * Z::BUF);
    if (tid < 2) odd_tile[tid] = 0u;
    block_prefix(a, group, R, pre, wave_sum, tid);
    const uint32_t blocks = __builtin_amdgcn_readfirstlane(pre[a.s.n_seqs]);
    if (blockIdx.y >= blocks) return;
    const uint32_t bi = blocks - 1u - blockIdx.y;
    uint32_t s;
    {
        uint32_t x = 0u, y = a.s.n_seqs - 1u;                // the last s with pre[s] <= bi
        while (x < y) {
            const uint32_t mid = (x + y + 1u) >> 1;
            if (pre[mid] <= bi) x = mid; else y = mid - 1u;
        }
        s = __builtin_amdgcn_readfirstlane(x);
    }
    uint32_t t0, t1;
    paged_rows(a.s, s, t0, t1);
    t0 = __builtin_amdgcn_readfirstlane(t0);
    t1 = __builtin_amdgcn_readfirstlane(t1);
    const uint32_t n_rows = (t1 - t0) * group;               // (< 2^31 * 2^16 would not fit: the launcher refuses n_tokens * n_heads >= 2^32)
    const uint32_t row0 = (bi - __builtin_amdgcn_readfirstlane(pre[s])) * R;
    const uint32_t row1 = n_rows - row0 < R ? n_rows : row0 + R;
    const int kv_len = (int)__builtin_amdgcn_readfirstlane(paged_kv_len(a.s, s));
    const int pos0 = kv_len - (int)(t1 - t0);                // position of the chunk's first token
    const int pmin = pos0 + (int)(row0 / group), pmax = pos0 + (int)((row1 - 1u) / group);
    // key tiles of the block: first tokens in front of the window of its first query, then up to its last query
    const uint32_t n_keys = pmax < 0 ? 0u : (uint32_t)pmax + 1u;
    const uint32_t lo_min = pmin > 0 ? paged_window_lo(a.window, (uint32_t)pmin) : 0u;
    const uint32_t first = lo_min / KT;
    const uint32_t sink = a.n_sink < lo_min ? a.n_sink : lo_min;
    const uint32_t su = (sink + KT - 1u) / KT;
    const uint32_t sink_tiles = su < first ? su : first;
    const uint32_t tiles = n_keys ? sink_tiles + (n_keys + KT - 1u) / KT - first : 0u;
    const uint32_t ta = (uint32_t)((uint64_t)blockIdx.z * tiles / n_split), tb = (uint32_t)((uint64_t)(blockIdx.z + 1u) * tiles / n_split);
    auto tile_key = [&](uint32_t t) { return (t < sink_tiles ? t : first + t - sink_tiles) * (uint32_t)KT; };

    // ---- this wavefront's rows
    const uint32_t wr0 = row0 + (uint32_t)w * 32u * NQ;
    const bool wave_has = wr0 < row1;
    const uint32_t wr1 = row1 < wr0 + 32u * NQ ? row1 : wr0 + 32u * NQ;
    const int wmin = wave_has ? pos0 + (int)(wr0 / group) : 0, wmax = wave_has ? pos0 + (int)((wr1 - 1u) / group) : -1;
    const int wlo_max = wmax > 0 ? (int)paged_window_lo(a.window, (uint32_t)wmax) : 0;     // window start of the last query
    const int wlo_min = wmin > 0 ? (int)paged_window_lo(a.window, (uint32_t)wmin) : 0;
    int pos[NQ], lo[NQ];
    uint32_t tok[NQ], head[NQ];
    bool real[NQ];
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        const uint32_t r = wr0 + 32u * q + (uint32_t)n32;
        real[q] = r < row1;
        const uint32_t rr = real[q] ? r : row0;
        tok[q] = rr / group;
        head[q] = kvh * group + rr - tok[q] * group;
        pos[q] = real[q] ? pos0 + (int)tok[q] : -1;
        lo[q] = pos[q] > 0 ? (int)paged_window_lo(a.window, (uint32_t)pos[q]) : 0;
        tok[q] += t0;
    }
    // ---- Q^T operands
    half8_t qh[F32C ? 1 : NQ][F32C ? 1 : D / 16], ql[PAIR ? NQ : 1][PAIR ? D / 16 : 1];
    float qf[F32C ? NQ : 1][F32C ? D / 2 : 1];
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        const uint64_t at = (uint64_t)tok[q] * a.q_stride + (uint64_t)head[q] * dr;
        if constexpr (F32C) {
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
                const uint32_t d = 8u * c + 4u * (uint32_t)hf;
                const bool ok = real[q] && d < dr;
                float4_t x;
                if constexpr (IOF16) {
                    const half4_t h = *reinterpret_cast<const half4_t*>(reinterpret_cast<const _Float16*>(a.q) + at + (ok ? d : 0u));
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[j] = (float)h[j];
                } else {
                    x = *reinterpret_cast<const float4_t*>(reinterpret_cast<const float*>(a.q) + at + (ok ? d : 0u));
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) qf[q][4 * c + j] = ok ? x[j] : 0.f;
            }
        } else {
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {
                const uint32_t d = 16u * c + 8u * (uint32_t)hf;
                const bool ok = real[q] && d < dr;
                if constexpr (IOF16) {
                    const half8_t x = *reinterpret_cast<const half8_t*>(reinterpret_cast<const _Float16*>(a.q) + at + (ok ? d : 0u));
#pragma unroll
                    for (int j = 0; j < 8; ++j) qh[q][c][j] = ok ? x[j] : (_Float16)0.f;
                } else {
                    const float* const src = reinterpret_cast<const float*>(a.q) + at + (ok ? d : 0u);
                    const float4_t x0 = *reinterpret_cast<const float4_t*>(src), x1 = *reinterpret_cast<const float4_t*>(src + 4);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float x = ok ? (j < 4 ? x0[j & 3] : x1[j & 3]) : 0.f;
                        const _Float16 hi = (_Float16)x;
                        qh[q][c][j] = hi;
                        ql[q][c][j] = (_Float16)(x - (float)hi);
                    }
                }
            }
        }
    }

    float16_t acc[DT32][NQ];
    float m[NQ], l[NQ];
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        m[q] = kMasked;
        l[q] = 0.f;
#pragma unroll
        for (int n = 0; n < DT32; ++n)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[n][q][e] = 0.f;
    }
    const float scale_l2 = a.scale * 1.44269504088896f;
    const float cap_l2 = a.softcap * 1.44269504088896f;
    const bool capped = a.softcap > 0.f;
    const float inv_cap_l2 = capped ? 1.0f / cap_l2 : 0.f;
    const float fac = capped ? 1.0f : scale_l2;              // scores are kept unscaled; the soft-cap leaves them in log2 units

    // ---- staging
    const uint32_t row_b = dr * Z::ES;
    const uint32_t chunk = (uint32_t)tid % Z::CPR, srow = (uint32_t)tid / Z::CPR;
    const bool chunk_ok = chunk * 16u < row_b;
    const uint64_t head_rows = (uint64_t)kvh << a.c.page_shift;
    const uint32_t slot_mask = (1u << a.c.page_shift) - 1u;
    const int32_t* const table = a.s.table + (uint64_t)s * a.s.table_stride;
    struct Pages {
        uint32_t p[KT / 16];
    };
    auto get_pages = [&](uint32_t t) {
        Pages r;
        const uint32_t kb = tile_key(t < tb ? t : tb - 1u);
#pragma unroll
        for (int i = 0; i < KT / 16; ++i) {
            const uint32_t key = kb + 16u * i;
            r.p[i] = (uint32_t)table[(key < n_keys ? key : n_keys - 1u) >> a.c.page_shift];
        }
        return r;
    };
    constexpr int NP = Z::NP < 1 ? 1 : Z::NP;
    u32x4 kraw[NP], vraw[NP];
    auto fetch = [&](const Pages& P, uint32_t t) {
        const uint32_t kb = tile_key(t);
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            const uint32_t sub = __builtin_amdgcn_readfirstlane(((uint32_t)(p * Z::RPP) + (uint32_t)w * (64u / Z::CPR)) / 16u);
            uint32_t page = P.p[0];
#pragma unroll
            for (int i = 1; i < KT / 16; ++i) page = sub == (uint32_t)i ? P.p[i] : page;
            if (page >= a.c.n_pages) page = 0u;
            const uint32_t key = kb + 16u * sub;
            const uint64_t off = (uint64_t)page * a.c.page_bytes + (head_rows + (key & slot_mask)) * row_b;
            const uint32_t lane_off = (((uint32_t)(p * Z::RPP) + srow) & 15u) * row_b + (chunk_ok ? chunk * 16u : 0u);
            kraw[p] = *reinterpret_cast<const u32x4*>(a.c.k + off + lane_off);
            vraw[p] = *reinterpret_cast<const u32x4*>(a.c.v + off + lane_off);
        }
    };
    // Rows no query of the block sees become zeros in V (their weights are zero, but 0 * NaN of a stale row is not), and a V
    // element that is not finite is reported: a query it is hidden from must not meet it (below).
    auto stage = [&](int buf, const Pages& P, uint32_t t) {
        uint8_t* const kl = lds + buf * Z::BUF;
        uint8_t* const vl = kl + KT * Z::KPITCH;
        const uint32_t kb = tile_key(t);
        bool part = kb + KT > (uint32_t)(pmin < 0 ? 0 : pmin + 1) ||
                    !(kb + KT <= a.n_sink || (a.window == 0u || kb >= paged_window_lo(a.window, (uint32_t)pmax)));
#pragma unroll
        for (int i = 0; i < KT / 16; ++i) part = part || P.p[i] >= a.c.n_pages;
        bool odd = false;
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            const uint32_t row = (uint32_t)(p * Z::RPP) + srow;
            u32x4 k = kraw[p], v = vraw[p];
            if (part) {
                uint32_t page = P.p[0];
#pragma unroll
                for (int i = 1; i < KT / 16; ++i) page = row / 16u == (uint32_t)i ? P.p[i] : page;
                const uint32_t key = kb + row;
                const bool ok = key < n_keys && (key >= lo_min || key < sink) && page < a.c.n_pages;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[i] = ok ? v[i] : 0u;
                    if constexpr (DT == kF32) odd = odd || (v[i] & 0x7F800000u) == 0x7F800000u;
                    else if constexpr (DT == kF16) odd = odd || (v[i] & 0x7C00u) == 0x7C00u || (v[i] & 0x7C000000u) == 0x7C000000u;
                    else odd = odd || (((v[i] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) != 0u;
                }
            }
            if (!chunk_ok) {
                k = u32x4{0u, 0u, 0u, 0u};
                v = k;
            }
            if (Z::RPP > KT && row >= (uint32_t)KT) continue;
            if constexpr (DT == kF8) {
                half2_t h[8];
                u32x4 o[2];
                auto widen = [&](const u32x4& x) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) e4m3x4_to_h2(x[i], h[2 * i], h[2 * i + 1]);
#pragma unroll
                    for (int i = 0; i < 8; ++i) o[i / 4][i % 4] = __builtin_bit_cast(uint32_t, h[i]);
                };
                widen(k);
                *reinterpret_cast<u32x4*>(kl + row * Z::KPITCH + chunk * 32u) = o[0];
                *reinterpret_cast<u32x4*>(kl + row * Z::KPITCH + chunk * 32u + 16u) = o[1];
                widen(v);
                *reinterpret_cast<u32x4*>(vl + row * Z::VPITCH + chunk * 32u) = o[0];
                *reinterpret_cast<u32x4*>(vl + row * Z::VPITCH + chunk * 32u + 16u) = o[1];
            } else {
                *reinterpret_cast<u32x4*>(kl + row * Z::KPITCH + chunk * 16u) = k;
                *reinterpret_cast<u32x4*>(vl + row * Z::VPITCH + chunk * 16u) = v;
            }
        }
        if (part && __any(odd)) odd_tile[buf] = t + 1u;
    };

    // ---- one tile
    auto compute = [&](int buf, const Pages& P, uint32_t t) {
        const uint8_t* const kl = lds + buf * Z::BUF;
        const uint8_t* const vl = kl + KT * Z::KPITCH;
        const int kb = (int)tile_key(t);
        bool ghost = false;
#pragma unroll
        for (int i = 0; i < KT / 16; ++i) ghost = ghost || P.p[i] >= a.c.n_pages;
        // seen by none of this wavefront's queries
        if (kb > wmax || (kb >= (int)a.n_sink && kb + KT <= wlo_min)) return;
        const bool full = kb + KT - 1 <= wmin && (kb >= wlo_max || kb + KT <= (int)a.n_sink) && !ghost;
        float16_t sc[NB][NQ];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int q = 0; q < NQ; ++q)
#pragma unroll
                for (int e = 0; e < 16; ++e) sc[b][q][e] = 0.f;
            const uint8_t* const krow = kl + (32 * b + n32) * Z::KPITCH + hf * 16;
            if constexpr (F32C) {
#pragma unroll
                for (int c = 0; c < D / 8; ++c) {
                    const float4_t k = *reinterpret_cast<const float4_t*>(krow + 32 * c);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int q = 0; q < NQ; ++q) sc[b][q] = __builtin_amdgcn_mfma_f32_32x32x2f32(k[j], qf[q][4 * c + j], sc[b][q], 0, 0, 0);
                }
            } else {
#pragma unroll
                for (int c = 0; c < D / 16; ++c) {
                    const half8_t k = *reinterpret_cast<const half8_t*>(krow + 32 * c);
#pragma unroll
                    for (int q = 0; q < NQ; ++q) {
                        sc[b][q] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qh[q][c], sc[b][q], 0, 0, 0);
                        if constexpr (PAIR) sc[b][q] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, ql[q][c], sc[b][q], 0, 0, 0);
                    }
                }
            }
        }
        if (capped) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int q = 0; q < NQ; ++q)
#pragma unroll
                    for (int e = 0; e < 16; ++e) sc[b][q][e] = softcap_l2(sc[b][q][e] * scale_l2, cap_l2, inv_cap_l2);
        }
        if (!full) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int key = kb + 32 * b + 8 * (e / 4) + 4 * hf + e % 4;
                    const bool there = P.p[2 * b + e / 8] < a.c.n_pages;
#pragma unroll
                    for (int q = 0; q < NQ; ++q) {
                        const bool seen = there && key <= pos[q] && (key >= lo[q] || key < (int)a.n_sink);
                        sc[b][q][e] = seen ? sc[b][q][e] : -__builtin_inff();
                    }
                }
        }
        float mx[NQ];
        bool raise = false;
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            mx[q] = sc[0][q][0];
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int e = 0; e < 16; ++e) mx[q] = fmaxf(mx[q], sc[b][q][e]);
            raise = raise || mx[q] * fac > m[q] + (kRaise + kBias);
        }
        if (__any(raise)) {
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
                const float mn = fmaxf(m[q], max_over_halves(mx[q]) * fac - kBias);
                const float corr = __builtin_amdgcn_exp2f(m[q] - mn);
                m[q] = mn;
                l[q] *= corr;
#pragma unroll
                for (int n = 0; n < DT32; ++n)
#pragma unroll
                    for (int e = 0; e < 16; ++e) acc[n][q][e] *= corr;
            }
        }
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int q = 0; q < NQ; ++q)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    sc[b][q][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[b][q][e], fac, -m[q]));
                    l[q] += sc[b][q][e];
                }
        if (!full && odd_tile[buf] == t + 1u) {
            // An infinity or NaN among the values of a tile that some of these queries see only in part: key by key, so that hidden
            // keys do not enter at all.
            for (int k = 0; k < KT; ++k) {
                const int e = 4 * ((k & 31) / 8) + (k & 3), src = ((k >> 2) & 1) * 32 + n32;
#pragma unroll
                for (int q = 0; q < NQ; ++q) {
                    float mine = 0.f;
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int x = 0; x < 16; ++x) mine = (b == k / 32 && x == e) ? sc[b][q][x] : mine;
                    const float p = __shfl(mine, src, kWave);
                    const int key = kb + k;
                    const bool seen = key <= pos[q] && (key >= lo[q] || key < (int)a.n_sink);   // (missing pages: 0 * 0)
#pragma unroll
                    for (int n = 0; n < DT32; ++n)
#pragma unroll
                        for (int x = 0; x < 16; ++x) {
                            const int d = 32 * n + 8 * (x / 4) + 4 * hf + x % 4;
                            float v;
                            if constexpr (F32C) v = *reinterpret_cast<const float*>(vl + k * Z::VPITCH + d * 4);
                            else v = (float)*reinterpret_cast<const _Float16*>(vl + k * Z::VPITCH + d * 2);
                            acc[n][q][x] = seen ? __builtin_fmaf(p, v, acc[n][q][x]) : acc[n][q][x];
                        }
                }
            }
            return;
        }
        if constexpr (F32C) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const uint8_t* const vrow = vl + (32 * b + 8 * (e / 4) + 4 * hf + e % 4) * Z::VPITCH + n32 * 4;
#pragma unroll
                    for (int n = 0; n < DT32; ++n) {
                        const float v = *reinterpret_cast<const float*>(vrow + 128 * n);
#pragma unroll
                        for (int q = 0; q < NQ; ++q) acc[n][q] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, sc[b][q][e], acc[n][q], 0, 0, 0);
                    }
                }
        } else {
            // lane's place in the transposing read: row 4 hf + (lane % 16) / 4 of eight-row steps, column group of its sixteen lanes
            const uint8_t* const vlane = vl + (4 * hf + (lane & 15) / 4) * Z::VPITCH + (16 * ((lane >> 4) & 1) + 4 * (lane & 3)) * 2;
#pragma unroll
            for (int kk = 0; kk < KT / 16; ++kk) {
                half8_t ph[NQ], pl[PAIR ? NQ : 1];
#pragma unroll
                for (int q = 0; q < NQ; ++q) {
                    uint32_t h[4], r[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float p0 = sc[kk / 2][q][8 * (kk % 2) + 2 * i], p1 = sc[kk / 2][q][8 * (kk % 2) + 2 * i + 1];
                        h[i] = __builtin_bit_cast(uint32_t, half2_t{(_Float16)p0, (_Float16)p1});
                        if constexpr (PAIR) r[i] = pack_f16_remainder(p0, p1, h[i]);
                    }
                    ph[q] = __builtin_bit_cast(half8_t, h);
                    if constexpr (PAIR) pl[q] = __builtin_bit_cast(half8_t, r);
                }
#pragma unroll
                for (int n = 0; n < DT32; ++n) {
                    const half4_t v0 = lds_read_tr16(reinterpret_cast<const _Float16*>(vlane + 16 * kk * Z::VPITCH + 64 * n));
                    const half4_t v1 = lds_read_tr16(reinterpret_cast<const _Float16*>(vlane + (16 * kk + 8) * Z::VPITCH + 64 * n));
                    const half8_t v = __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
                    for (int q = 0; q < NQ; ++q) {
                        acc[n][q] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, ph[q], acc[n][q], 0, 0, 0);
                        if constexpr (PAIR) acc[n][q] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pl[q], acc[n][q], 0, 0, 0);
                    }
                }
            }
        }
    };

    if (ta < tb) {
        Pages p0 = get_pages(ta), p1 = get_pages(ta + 1u);
        fetch(p0, ta);
        stage(0, p0, ta);
        for (uint32_t t = ta; t < tb; ++t) {
            const int buf = (int)((t - ta) & 1u);
            __syncthreads();                                   // tile t staged by all; tile t - 1 no longer read
            const Pages p2 = get_pages(t + 2u);
            if (t + 1u < tb) fetch(p1, t + 1u);
            if (wave_has) compute(buf, p0, t);
            if (t + 1u < tb) stage(buf ^ 1, p1, t + 1u);
            p0 = p1;
            p1 = p2;
        }
    }

    // ---- output
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        const float L = xor32_sum(l[q]);
        if (!real[q]) continue;
        const float inv = n_split > 1u ? 1.0f : L != 0.f ? 1.0f / L : 0.f;
        const uint64_t row = ((uint64_t)tok[q] * a.n_heads + head[q]) * n_split + blockIdx.z;
        const uint64_t at = (uint64_t)tok[q] * a.o_stride + (uint64_t)head[q] * dr;
        if (n_split > 1u && hf == 0) { a.scratch_max[row] = m[q]; a.scratch_sum[row] = L; }
#pragma unroll
        for (int n = 0; n < DT32; ++n)
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const uint32_t d = 32u * n + 8u * b + 4u * (uint32_t)hf;
                if (d >= dr) continue;
                float4_t v;
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = acc[n][q][4 * b + j] * inv;
                if (n_split > 1u) {
                    *reinterpret_cast<float4_t*>(a.scratch_out + row * dr + d) = v;
                } else if constexpr (IOF16) {
                    half4_t h;
#pragma unroll
                    for (int j = 0; j < 4; ++j) h[j] = (_Float16)v[j];
                    *reinterpret_cast<half4_t*>(reinterpret_cast<_Float16*>(a.o) + at + d) = h;
                } else {
                    *reinterpret_cast<float4_t*>(reinterpret_cast<float*>(a.o) + at + d) = v;
                }
            }
    }
}

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

namespace {

template <int DT, int D, bool IOF16, int NQ, int KT, int MINW>
hipError_t launch_pre(const PagedAttnLaunch& L, hipStream_t stream) {
    using Z = PreShape<DT, D, KT>;
    constexpr uint64_t R = 128u * NQ;
    const uint64_t group = L.n_heads / L.c.n_kv_heads;
    // a sequence's last block may be ragged: at most one block more per sequence that has rows
    const uint64_t with_rows = L.s.n_seqs < L.s.n_tokens ? L.s.n_seqs : L.s.n_tokens;
    uint64_t blocks = L.s.n_tokens * group / R + with_rows;
    if (blocks > L.s.n_tokens * group) blocks = L.s.n_tokens * group;
    if (blocks > 65535u * 4096ull) return hipErrorInvalidValue;
    // split over the keys: as long as the card has room, at least four tiles per part
    const uint64_t likely = (L.s.n_tokens * group + R - 1u) / R * L.c.n_kv_heads;
    const uint64_t room = 256u * MINW;
    uint64_t keys = L.max_kv;
    if (L.window != 0u && (uint64_t)L.window + L.n_sink + R + 2u * KT < keys) keys = (uint64_t)L.window + L.n_sink + R + 2u * KT;
    uint64_t n = room / likely;
    if (n > keys / (4u * KT)) n = keys / (4u * KT);
    const uint64_t fits = L.scratch_rows / ((uint64_t)L.s.n_tokens * L.n_heads);
    if (n > fits) n = fits;
    if (n > 64u) n = 64u;
    if (n == 0u) n = 1u;
    hipLaunchKernelGGL((paged_prefill_kernel<DT, D, IOF16, NQ, KT, MINW>), dim3(L.c.n_kv_heads, (uint32_t)blocks, (uint32_t)n), dim3(256),
                       2u * Z::BUF + (L.s.n_seqs + 1u) * 4u, stream, L, (uint32_t)n);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || n == 1u) return e;
    const uint32_t per = 256u / (L.c.head_dim / 4u);
    const uint64_t rows = (uint64_t)L.s.n_tokens * L.n_heads;
    hipLaunchKernelGGL(paged_rows_merge_kernel, dim3((uint32_t)((rows + per - 1u) / per)), dim3(256), 0, stream, L, (uint32_t)n);
    return hipGetLastError();
}

template <int DT, bool IOF16>
hipError_t launch_dim(const PagedAttnLaunch& L, hipStream_t stream) {
    const uint32_t d = L.c.head_dim;
    if constexpr (DT == kF32) {
        if (d <= 64u) return launch_pre<DT, 64, IOF16, 1, 32, 2>(L, stream);
        if (d <= 128u) return launch_pre<DT, 128, IOF16, 1, 32, 2>(L, stream);
        return launch_pre<DT, 256, IOF16, 1, 32, 1>(L, stream);
    } else {
        // two row blocks per wavefront halve the LDS reads per product: for enough rows to fill the card that way
        const bool many = (uint64_t)L.s.n_tokens * L.n_heads >= 256u * 256u;
        if (d <= 64u) return IOF16 && many ? launch_pre<DT, 64, IOF16, IOF16 ? 2 : 1, 64, 2>(L, stream) : launch_pre<DT, 64, IOF16, 1, 64, 2>(L, stream);
        if (d <= 128u) return IOF16 && many ? launch_pre<DT, 128, IOF16, IOF16 ? 2 : 1, 64, IOF16 ? 1 : 2>(L, stream) : launch_pre<DT, 128, IOF16, 1, 64, 2>(L, stream);
        return launch_pre<DT, 256, IOF16, 1, 32, 1>(L, stream);
    }
}

}  // namespace

hipError_t launch_paged_prefill(const PagedAttnLaunch& L, hipStream_t stream) {
    if ((uint64_t)L.s.n_tokens * L.n_heads > 0xFFFFFFFFull) return hipErrorInvalidValue;
    if (L.c.dtype == kF8) return L.io_f16 ? launch_dim<kF8, true>(L, stream) : launch_dim<kF8, false>(L, stream);
    if (L.c.dtype == kF16) return L.io_f16 ? launch_dim<kF16, true>(L, stream) : launch_dim<kF16, false>(L, stream);
    return L.io_f16 ? launch_dim<kF32, true>(L, stream) : launch_dim<kF32, false>(L, stream);
}

}  // namespace vfkv
