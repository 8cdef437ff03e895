// Decode attention over the paged cache: one token per sequence, a batch of sequences of any lengths.
//
// o = sum_j softmax_j(scale q.k_j) v_j per head; bound by reading K and V once (4 flop per element and query head against 1, 2 or 4
// bytes), so the kernel is built around keeping loads in flight on every CU whatever the lengths are:
//
//   - The keys of ALL sequences, cut into units of 16 * SUB aligned positions (first tokens, then the window), with a few units in
//     front of each sequence for what beginning it costs, are one line of U units per KV head.  Workgroup w of N owns units [w U / N, (w + 1) U / N): every workgroup has the same work to one unit, a
//     long sequence is spread over many workgroups and short ones are packed.  A workgroup's range touches at most two
//     sequences partly (its first and its last); those parts leave unnormalised sums that paged_merge_kernel joins, sequences
//     inside the range are written directly.  The lengths are device data, so each workgroup finds its range itself
//     (a prefix sum over the batch in LDS).
//   - The four wavefronts of a workgroup take the units of a sequence in turn.  A 16-key tile lies in one page (page sizes are
//     multiples of 16), so a page number is one scalar load, requested two units ahead; K and V rows go from memory to
//     registers one unit ahead.
//   - Both products run on the matrix cores, transposed, so that no register changes lanes in between:
//       S^T[key, col] = K Q^T: A = K rows as loaded (FP8 widened exactly), B = Q^T.  Columns 0-7 hold f16(q'), columns 8-15
//         f16(q' - f16(q')) of the same heads (q' = q times a power of two): the sum of both columns has f32-level accuracy.
//       O^T[d, col] += V^T P^T: B = P as the score tile left it (a lane holds four consecutive keys of one column, which is what
//         the operand wants when the contraction runs over the keys in that order), columns 0-7 f16(p), 8-15 the remainder.
//         A = V^T: a lane loads D / 16 columns of its four keys per tile and turns that small matrix with byte permutes
//         in its own registers -- no LDS, no barrier.
//     F32 caches use the f32 matrix instruction with the same ownership; nothing needs turning there.
// Measured, one layer (copy rate of the card: 5.2 TB/s): 48 sequences of 17-8 193 keys, FP8, 32 / 8 / 128: 80.6 us = 4.8 TB/s; 12 windows
// of 4 096 keys, F16, 16 / 8 / 256, soft-capped: 77.1 us = 5.0 TB/s; one sequence of 65 536 keys: 25.8 us for the worker (5.2 TB/s) and
// 6.0 us for the join; one of 200 keys 6.5 us (the chain length -> page -> rows -> join of the wavefronts).  Rows of 512, 48 sequences of
// up to 8 000 keys, 8 KV heads: FP8 310 us = 5.1 TB/s, F16 538 us = 5.8 TB/s.  F32 pages, the first batch: 291 us = 5.3 TB/s, with 19
// registers spilled (6 at rows of 256).
//
//   - The running maximum is only raised when a score exceeds it by 2^8 (paged.h), so that the accumulators are rescaled a few times
//     per sequence instead of once per unit.
#include "device_utils.h"
#include "paged.h"

namespace vfkv {

namespace {

constexpr int kDecWaves = 4;
// Query heads of a KV head per workgroup: a larger group is cut into slices of eight, each of which reads the keys again (48 sequences of
// 17-8 193 keys, FP8, 64 / 4 heads 72.9 us, 32 / 4 50.5; 12 / 1 29.0, 8 / 1 23.5).
constexpr int kDecHeads = 8;
// What beginning a sequence costs a workgroup (queries, page numbers, the join of its wavefronts), in units: it stands in front of
// the sequence's own units in the line.  Without it 124 sequences of 7 to 11 keys went to 16 workgroups of eight each.
constexpr uint32_t kBegin = 2u * kDecWaves;

template <int DT, int D, int SUB_>
struct DecShape {
    static constexpr int ES = DT == kF32 ? 4 : DT == kF16 ? 2 : 1;
    static constexpr int SUB = SUB_;                     // 16-key tiles per unit
    static constexpr int UK = 16 * SUB;                  // keys per unit
    static constexpr int SHIFT = SUB == 1 ? 4 : SUB == 2 ? 5 : 6;
    static_assert(UK == 1 << SHIFT, "units are powers of two");
    static constexpr int KE = 16 / ES;                   // elements of a 16-byte piece of a K row
    static constexpr int KL = D / (4 * KE);              // pieces per lane and row: piece x of lane group g is elements (4 x + g) KE ..
    static constexpr int NT = D / 16;                    // d-tiles = V elements per lane and key
    static constexpr int PE = NT < KE ? NT : KE;         // elements of a V piece: piece y of lane r is elements (16 y + r) PE ..
    static constexpr int VP = NT / PE;                   // V pieces
    static constexpr int PW = PE * ES / 4;               // dwords of a V piece
    static constexpr int VW = VP * PW;                   // V dwords per lane and key
    // Rows of 512: two units in registers beside the sums and queries do not fit (F16: 387 registers spilled).  One, whose K half is
    // requested again when the scores are there and whose V half when the outputs are.  (FP8, where two fit through copies to the
    // accumulation registers, 64 sequences of 200-600 keys: two / one 48.2 / 45.3 us.)
    static constexpr bool ONE = D == 512;
};

// Units of a sequence: first tokens, then the window of the query at position len - 1, as far as there are rows (n keys).
struct SeqUnits {
    uint32_t n, lo, sink, sink_units, first, units;
};
__device__ __forceinline__ SeqUnits seq_units(const PagedAttnLaunch& a, uint32_t len, uint32_t uk_shift) {
    const uint32_t uk = 1u << uk_shift, n = len < a.s.limit ? len : a.s.limit, n_sink = a.n_sink;
    const uint32_t lo = len ? paged_window_lo(a.window, len - 1u) : 0u;
    SeqUnits r;
    r.n = n;
    r.lo = lo < n ? lo : n;
    r.sink = n_sink < r.lo ? n_sink : r.lo;
    r.first = r.lo >> uk_shift;
    const uint32_t su = (r.sink + uk - 1u) >> uk_shift;
    r.sink_units = su < r.first ? su : r.first;         // what reaches the window's first unit belongs to it
    r.units = n ? r.sink_units + ((n + uk - 1u) >> uk_shift) - r.first : 0u;
    return r;
}

// Workgroups that share a line of U units: the launch's, or as many as get two units per wavefront besides a sequence's beginning.
// Never more than U, so that no range is empty; 0 for an empty batch.
__device__ __forceinline__ uint32_t used_wgs(uint32_t U, uint32_t n_wg) {
    const uint32_t most = (U + kBegin + 2u * kDecWaves - 1u) / (kBegin + 2u * kDecWaves);
    return most < n_wg ? most : n_wg;
}

// floor(a / b) for a < 2^41, b < 2^32 through f64: a quotient that is not whole is at least 2^-41 of itself away from the next whole
// number, the division rounds by 2^-53.  (The 64-bit integer division is some hundred instructions.)
__device__ __forceinline__ uint32_t div_floor(uint64_t a, uint32_t b) { return (uint32_t)((double)a / (double)b); }

__device__ __forceinline__ float max_over_groups(float x) {   // over lanes with the same lane & 15
    float y = x;
    swap16(x, y);
    x = fmaxf(x, y);
    y = x;
    swap32(x, y);
    return fmaxf(x, y);
}
__device__ __forceinline__ float sum_over_groups(float x) { return xor32_sum(xor16_sum(x)); }
__device__ __forceinline__ float ror8_sum(float x) { return x + dpp_f<kDppRor8>(x); }   // columns c and c + 8

}  // namespace

// Length of a sequence in the line of units.
__device__ __forceinline__ uint32_t line_units(uint32_t units) { return units ? units + kBegin : 0u; }

// Prefix sums of the line: pre[s] for s <= n_seqs, by the whole workgroup.
template <int SHIFT>
__device__ __forceinline__ void unit_prefix(const PagedAttnLaunch& a, uint32_t* pre, uint32_t* wave_sum, int tid) {
    const int lane = tid & 63, w = tid >> 6;
    uint32_t carry = 0u;
    for (uint32_t base = 0; base < a.s.n_seqs; base += 256u) {
        const uint32_t s = base + (uint32_t)tid;
        uint32_t x = s < a.s.n_seqs ? line_units(seq_units(a, paged_kv_len(a.s, s), SHIFT).units) : 0u;
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
        for (int i = 0; i < kDecWaves; ++i) {
            if (i < w) before += wave_sum[i];
            carry += wave_sum[i];
        }
        if (s < a.s.n_seqs) pre[s] = before + x - mine;
        __syncthreads();
    }
    if (tid == 0) pre[a.s.n_seqs] = carry;
    __syncthreads();
}

template <int DT, int D, int SUB>
__global__ __launch_bounds__(256, D >= 256 ? 1 : 2) void paged_decode_kernel(PagedAttnLaunch a, uint32_t n_wg, uint32_t slices, uint32_t direct) {
    using Z = DecShape<DT, D, SUB>;
    constexpr int OP = D + 4;                                            // pitch of an output row in LDS
    __shared__ __attribute__((aligned(16))) float o_lds[kDecWaves][kDecHeads][OP];
    __shared__ float m_lds[kDecWaves][kDecHeads], l_lds[kDecWaves][kDecHeads];
    __shared__ uint32_t wave_sum[kDecWaves];
    extern __shared__ uint32_t pre[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n16 = lane & 15, g = lane >> 4, col = n16 & 7;
    const bool is_lo = n16 >= 8;
    const uint32_t wg = blockIdx.y;
    const uint32_t kvh = blockIdx.x / slices, slice = blockIdx.x - kvh * slices;
    const uint32_t group = a.n_heads / a.c.n_kv_heads;
    const uint32_t h0 = kvh * group + slice * kDecHeads;
    const uint32_t heads = group - slice * kDecHeads < (uint32_t)kDecHeads ? group - slice * kDecHeads : (uint32_t)kDecHeads;
    const uint32_t dr = a.c.head_dim;
    auto no_keys = [&](uint32_t s) {                                      // a sequence without a key: zeros
        for (uint32_t e = tid; e < heads * dr; e += 256u) {
            const uint64_t at = (uint64_t)s * a.o_stride + (uint64_t)h0 * dr + e;
            if (a.io_f16) reinterpret_cast<_Float16*>(a.o)[at] = (_Float16)0.f; else reinterpret_cast<float*>(a.o)[at] = 0.f;
        }
    };
    uint32_t u0 = 0u, u1, s_first, s_end = a.s.n_seqs;
    if (direct) {
        s_first = wg;
        s_end = wg + 1u;
        u1 = line_units(seq_units(a, __builtin_amdgcn_readfirstlane(paged_kv_len(a.s, wg)), Z::SHIFT).units);
        if (u1 == 0u) { no_keys(wg); return; }
    } else {
        unit_prefix<Z::SHIFT>(a, pre, wave_sum, tid);
        const uint32_t U = pre[a.s.n_seqs];
        for (uint32_t s = wg; s < a.s.n_seqs; s += n_wg)
            if (pre[s + 1u] == pre[s]) no_keys(s);
        const uint32_t n_eff = used_wgs(U, n_wg);
        if (wg >= n_eff) return;
        u0 = __builtin_amdgcn_readfirstlane(div_floor((uint64_t)wg * U, n_eff));
        u1 = __builtin_amdgcn_readfirstlane(div_floor((uint64_t)(wg + 1u) * U, n_eff));
        uint32_t x = 0u, y = a.s.n_seqs - 1u;                            // the last s with pre[s] <= u0 (it has units)
        while (x < y) {
            const uint32_t mid = (x + y + 1u) >> 1;
            if (pre[mid] <= u0) x = mid; else y = mid - 1u;
        }
        s_first = __builtin_amdgcn_readfirstlane(x);
    }
    const float scale_l2 = a.scale * 1.44269504088896f;
    const float cap_l2 = a.softcap * 1.44269504088896f;
    const float inv_cap_l2 = a.softcap > 0.f ? 1.0f / cap_l2 : 0.f;
    // lane parts of the row addresses (pieces past a narrower head read its first piece again: they meet zeros of q, or are not stored)
    const uint32_t row_b = dr * Z::ES;
    uint32_t koff[Z::KL], voff[Z::VP];
#pragma unroll
    for (int x = 0; x < Z::KL; ++x) {
        const uint32_t e = (uint32_t)(4 * x + g) * Z::KE;
        koff[x] = (uint32_t)n16 * row_b + (e < dr ? e * Z::ES : 0u);
    }
#pragma unroll
    for (int y = 0; y < Z::VP; ++y) {
        const uint32_t e = (uint32_t)(16 * y + n16) * Z::PE;
        voff[y] = 4u * (uint32_t)g * row_b + (e < dr ? e * Z::ES : 0u);
    }
    const uint64_t head_b = (uint64_t)kvh << a.c.page_shift;             // rows in front of this head's in a page
    const uint32_t slot_mask = (1u << a.c.page_shift) - 1u;

    struct Stage {
        u32x4 k[SUB][Z::KL];
        uint32_t v[SUB][4][Z::VW];
    };
    struct Pages {
        uint32_t p[SUB];
    };

    for (uint32_t s = s_first; s < s_end; ++s) {
        const uint32_t ps = direct ? 0u : __builtin_amdgcn_readfirstlane(pre[s]), pe = direct ? u1 : __builtin_amdgcn_readfirstlane(pre[s + 1u]);
        if (ps >= u1) break;
        if (ps == pe) continue;
        const SeqUnits Q = seq_units(a, __builtin_amdgcn_readfirstlane(paged_kv_len(a.s, s)), Z::SHIFT);
        // this range's part of the sequence, units [ua, ub)
        const uint32_t la = (ps > u0 ? ps : u0) - ps, lb = (pe < u1 ? pe : u1) - ps;
        const uint32_t ua = la > kBegin ? la - kBegin : 0u, ub = lb > kBegin ? lb - kBegin : 0u;
        if (ua >= ub) continue;
        const int32_t* const table = a.s.table + (uint64_t)s * a.s.table_stride;

        // ---- q' as the B operand of the first product
        half8_t qb[DT == kF32 ? 1 : D / 32];
        float qf[DT == kF32 ? D / 4 : 1];
        float fac = 1.0f;                                                 // of the scores, to log2 units
        {
            const bool there = (uint32_t)col < heads && (DT != kF32 || !is_lo);
            const uint64_t qrow = (uint64_t)s * a.q_stride + (uint64_t)(h0 + (there ? (uint32_t)col : 0u)) * dr;
            auto load8 = [&](uint32_t d, float* out, int n, float by) {   // n = 4 or 8 elements of the head's row, times `by`
                const bool ok = there && d < dr;
                const uint64_t at = qrow + (ok ? d : 0u);
                for (int j = 0; j < n; j += 4) {
                    float x[4];
                    if (a.io_f16) {
                        const half4_t h = *reinterpret_cast<const half4_t*>(reinterpret_cast<const _Float16*>(a.q) + at + j);
                        for (int i = 0; i < 4; ++i) x[i] = (float)h[i];
                    } else {
                        const float4_t f = *reinterpret_cast<const float4_t*>(reinterpret_cast<const float*>(a.q) + at + j);
                        for (int i = 0; i < 4; ++i) x[i] = f[i];
                    }
                    for (int i = 0; i < 4; ++i) out[j + i] = ok ? x[i] * by : 0.f;
                }
            };
            if constexpr (DT == kF32) {
#pragma unroll
                for (int x = 0; x < Z::KL; ++x) load8((uint32_t)(4 * x + g) * 4u, &qf[4 * x], 4, scale_l2);
            } else {
                // times the power of two that brings the row's largest element to [0.5, 1): value + remainder hold every element to
                // 2^-23 of that, whatever the row's size
                float x[D / 32][8], top = 0.f;
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    constexpr int PER = Z::KE / 8;                       // operands per piece
                    load8((uint32_t)(4 * (c / PER) + g) * Z::KE + 8u * (uint32_t)(c % PER), x[c], 8, 1.0f);
#pragma unroll
                    for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(x[c][j]));
                }
                const int e = __builtin_amdgcn_frexp_expf(max_over_groups(top));
                fac = fmaxf(__builtin_ldexpf(scale_l2, e), 1e-37f);       // (not 0: -inf * 0 of a hidden key would be NaN)
#pragma unroll
                for (int c = 0; c < D / 32; ++c)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float y = __builtin_ldexpf(x[c][j], -e);
                        const _Float16 hi = (_Float16)y;
                        qb[c][j] = is_lo ? (_Float16)(y - (float)hi) : hi;
                    }
            }
        }

        float4_t acc[Z::NT];
#pragma unroll
        for (int n = 0; n < Z::NT; ++n) acc[n] = float4_t{0.f, 0.f, 0.f, 0.f};
        float m = kNoScore, l = 0.f;                                     // l: this lane's keys only, summed at the end
        bool far = false;                                                // some head is far out: its products are rounded before they are compared

        auto unit_key = [&](uint32_t u) { return (u < Q.sink_units ? u : Q.first + u - Q.sink_units) * (uint32_t)Z::UK; };
        auto get_pages = [&](uint32_t u) {
            Pages r;
            const uint32_t kb = unit_key(u < ub ? u : ub - 1u);
#pragma unroll
            for (int t = 0; t < SUB; ++t) {
                const uint32_t key = kb + 16u * t;
                r.p[t] = (uint32_t)table[(key < Q.n ? key : Q.n - 1u) >> a.c.page_shift];
            }
            return r;
        };
        auto load = [&](Stage& st, const Pages& P, uint32_t u, bool ks = true, bool vs = true) {   // past the end: the last unit again, from the cache
            const uint32_t kb = unit_key(u < ub ? u : ub - 1u);
#pragma unroll
            for (int t = 0; t < SUB; ++t) {
                const uint32_t key = kb + 16u * t;
                const uint32_t page = P.p[t] < a.c.n_pages ? P.p[t] : 0u;
                // (a tile past the last key reads the page of the last key, inside the page: masked below)
                const uint64_t off = (uint64_t)page * a.c.page_bytes + (head_b + (key & slot_mask)) * row_b;
                const uint8_t* const kp = a.c.k + off;
                const uint8_t* const vp = a.c.v + off;
#pragma unroll
                for (int x = 0; x < Z::KL; ++x)
                    if (ks) st.k[t][x] = *reinterpret_cast<const u32x4*>(kp + koff[x]);
                if (!vs) continue;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int y = 0; y < Z::VP; ++y) {
                        const uint8_t* const src = vp + (voff[y] + (uint32_t)i * row_b);
                        if constexpr (Z::PW == 4) {
                            const u32x4 x = *reinterpret_cast<const u32x4*>(src);
#pragma unroll
                            for (int e = 0; e < 4; ++e) st.v[t][i][4 * y + e] = x[e];
                        } else if constexpr (Z::PW == 2) {
                            const u32x2 x = *reinterpret_cast<const u32x2*>(src);
                            st.v[t][i][2 * y] = x[0];
                            st.v[t][i][2 * y + 1] = x[1];
                        } else {
                            st.v[t][i][y] = *reinterpret_cast<const uint32_t*>(src);
                        }
                    }
            }
        };
        auto compute = [&](Stage& st, const Pages& P, uint32_t u, auto&& scored) {
            const uint32_t kb = unit_key(u);
            bool full = kb + (uint32_t)Z::UK <= Q.n && (kb >= Q.lo || kb + (uint32_t)Z::UK <= Q.sink);
#pragma unroll
            for (int t = 0; t < SUB; ++t) full = full && P.p[t] < a.c.n_pages;
            float x[SUB][4];
#pragma unroll
            for (int t = 0; t < SUB; ++t) {
                float4_t sc = {0.f, 0.f, 0.f, 0.f};
                if constexpr (DT == kF32) {
#pragma unroll
                    for (int p = 0; p < Z::KL; ++p) {
                        const float4_t kf = __builtin_bit_cast(float4_t, st.k[t][p]);   // (whole: a bit_cast of one element reads element 0)
#pragma unroll
                        for (int j = 0; j < 4; ++j) sc = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[j], qf[4 * p + j], sc, 0, 0, 0);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[t][i] = sc[i];
                } else {
#pragma unroll
                    for (int c = 0; c < D / 32; ++c) {
                        half8_t ka;
                        if constexpr (DT == kF16) {
                            ka = __builtin_bit_cast(half8_t, st.k[t][c]);
                        } else {
                            half2_t h[4];
                            e4m3x4_to_h2(st.k[t][c / 2][2 * (c % 2)], h[0], h[1]);
                            e4m3x4_to_h2(st.k[t][c / 2][2 * (c % 2) + 1], h[2], h[3]);
                            ka = __builtin_bit_cast(half8_t, h);
                        }
                        sc = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qb[c], sc, 0, 0, 0);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[t][i] = ror8_sum(sc[i]);
                }
            }
            scored();                                                    // (K is used up)
            float to_l2 = fac;
            if (a.softcap > 0.f) {
                to_l2 = 1.0f;                                            // (the soft-cap leaves log2 units)
#pragma unroll
                for (int t = 0; t < SUB; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[t][i] = paged_softcap_l2(x[t][i] * fac, cap_l2, inv_cap_l2);
            }
            bool rounded = false;
            auto round_products = [&](bool mine) {                       // of this lane's head; the others keep theirs
                const float by = mine ? fac : 1.0f;
                to_l2 = mine ? 1.0f : to_l2;
                rounded = rounded || mine;
#pragma unroll
                for (int t = 0; t < SUB; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[t][i] *= by;
            };
            if (DT != kF32 && far) round_products(paged_far(m));         // (F32: fac is 1; far is never set with a soft-cap)
            if (!full) {
#pragma unroll
                for (int t = 0; t < SUB; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t key = kb + 16u * t + 4u * (uint32_t)g + (uint32_t)i;
                        const bool seen = key < Q.n && (key >= Q.lo || key < Q.sink) && P.p[t] < a.c.n_pages;
                        x[t][i] = seen ? x[t][i] : -__builtin_inff();
#pragma unroll
                        for (int e = 0; e < Z::VW; ++e) st.v[t][i][e] = seen ? st.v[t][i][e] : 0u;   // 0 * NaN of a stale row is NaN
                    }
            }
            float mx = x[0][0];
#pragma unroll
            for (int t = 0; t < SUB; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) mx = fmaxf(mx, x[t][i]);
            if (__any(mx * to_l2 - m > kRaise + kBias<DT>)) {
                const float mn = fmaxf(m, max_over_groups(mx * to_l2) - kBias<DT>);
                if (DT != kF32 && !(a.softcap > 0.f)) {
                    far = __any(paged_far(mn));
                    if (far) round_products(paged_far(mn) && !rounded);
                }
                const float corr = __builtin_amdgcn_exp2f(m - mn);
                m = mn;
                l *= corr;
#pragma unroll
                for (int n = 0; n < Z::NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[n][i] *= corr;
            }
#pragma unroll
            for (int t = 0; t < SUB; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[t][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[t][i], to_l2, -m));
                    l += x[t][i];
                }
            if constexpr (DT == kF32) {
#pragma unroll
                for (int t = 0; t < SUB; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int n = 0; n < Z::NT; ++n)
                            acc[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, st.v[t][i][n]), x[t][i], acc[n], 0, 0, 0);
            } else {
                uint32_t p[SUB][2];
#pragma unroll
                for (int t = 0; t < SUB; ++t)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t hi = __builtin_bit_cast(uint32_t, half2_t{(_Float16)x[t][2 * i], (_Float16)x[t][2 * i + 1]});
                        const uint32_t lo = pack_f16_remainder(x[t][2 * i], x[t][2 * i + 1], hi);
                        p[t][i] = is_lo ? lo : hi;
                    }
                // dword e of a key's V piece against the same dword of its neighbour: columns side by side -> keys side by side
                auto turned = [&](int t, int n, int pair) -> uint32_t {   // V^T operand dword: keys 2 pair, 2 pair + 1 of tile t, d-tile n
                    const uint32_t* const ka = st.v[t][2 * pair];
                    const uint32_t* const kb2 = st.v[t][2 * pair + 1];
                    if constexpr (DT == kF16) {
                        return __builtin_amdgcn_perm(kb2[n / 2], ka[n / 2], n % 2 ? 0x07060302u : 0x05040100u);
                    } else {
                        const uint32_t c = __builtin_amdgcn_perm(kb2[n / 4], ka[n / 4], n % 4 >= 2 ? 0x07030602u : 0x05010400u);
                        const half2_t h = n % 2 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)c, 1.0f, true)
                                                : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)c, 1.0f, false);
                        return __builtin_bit_cast(uint32_t, h);
                    }
                };
                if constexpr (SUB % 2 == 0) {
#pragma unroll
                    for (int t = 0; t < SUB; t += 2) {
                        const half8_t pb = __builtin_bit_cast(half8_t, u32x4{p[t][0], p[t][1], p[t + 1][0], p[t + 1][1]});
#pragma unroll
                        for (int n = 0; n < Z::NT; ++n) {
                            const half8_t va = __builtin_bit_cast(half8_t, u32x4{turned(t, n, 0), turned(t, n, 1), turned(t + 1, n, 0), turned(t + 1, n, 1)});
                            acc[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pb, acc[n], 0, 0, 0);
                        }
                    }
                } else {
#pragma unroll
                    for (int t = 0; t < SUB; ++t) {
                        const half4_t pb = __builtin_bit_cast(half4_t, u32x2{p[t][0], p[t][1]});
#pragma unroll
                        for (int n = 0; n < Z::NT; ++n) {
                            const half4_t va = __builtin_bit_cast(half4_t, u32x2{turned(t, n, 0), turned(t, n, 1)});
                            acc[n] = __builtin_amdgcn_mfma_f32_16x16x16f16(va, pb, acc[n], 0, 0, 0);
                        }
                    }
                }
            }
        };

        if (ua + (uint32_t)w < ub) {
            if constexpr (Z::ONE) {
                Stage st;
                uint32_t u = ua + (uint32_t)w;
                Pages p0 = get_pages(u), p1 = get_pages(u + kDecWaves);
                load(st, p0, u);
                for (;;) {
                    const Pages p2 = get_pages(u + 2u * kDecWaves);
                    compute(st, p0, u, [&] { load(st, p1, u + kDecWaves, true, false); });
                    load(st, p1, u + kDecWaves, false, true);
                    u += kDecWaves;
                    if (u >= ub) break;
                    p0 = p1;
                    p1 = p2;
                }
            } else {
                Stage st0, st1;
                uint32_t u = ua + (uint32_t)w;
                Pages p0 = get_pages(u), p1 = get_pages(u + kDecWaves);
                load(st0, p0, u);
                for (;;) {
                    Pages p2 = get_pages(u + 2u * kDecWaves);
                    load(st1, p1, u + kDecWaves);
                    compute(st0, p0, u, [] {});
                    u += kDecWaves;
                    if (u >= ub) break;
                    p0 = p2;
                    p2 = get_pages(u + 2u * kDecWaves);
                    load(st0, p0, u + kDecWaves);
                    compute(st1, p1, u, [] {});
                    u += kDecWaves;
                    if (u >= ub) break;
                    p1 = p2;
                }
            }
        }

        // ---- the four wavefronts' parts joined through LDS
        l = sum_over_groups(l);
        if constexpr (DT != kF32) {
#pragma unroll
            for (int n = 0; n < Z::NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[n][i] = ror8_sum(acc[n][i]);
        }
        if (!is_lo) {
#pragma unroll
            for (int y = 0; y < Z::VP; ++y)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < Z::PE; j += 4) {
                        float4_t v;
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] = acc[y * Z::PE + j + e][i];
                        *reinterpret_cast<float4_t*>(&o_lds[w][col][(16 * y + 4 * g + i) * Z::PE + j]) = v;
                    }
            if (g == 0) { m_lds[w][col] = m; l_lds[w][col] = l; }
        }
        __syncthreads();
        const bool whole = ua == 0u && ub == Q.units;
        const uint64_t part = (uint64_t)wg * 2u + (s == s_first ? 0u : 1u);
        for (uint32_t e = tid; e < heads * (D / 4); e += 256u) {
            const uint32_t h = e / (D / 4), d = (e % (D / 4)) * 4u;
            float M = m_lds[0][h];
#pragma unroll
            for (int i = 1; i < kDecWaves; ++i) M = fmaxf(M, m_lds[i][h]);
            float L = 0.f;
            float4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < kDecWaves; ++i) {
                const float f = __builtin_amdgcn_exp2f(m_lds[i][h] - M);
                L = __builtin_fmaf(l_lds[i][h], f, L);
                const float4_t v = *reinterpret_cast<const float4_t*>(&o_lds[i][h][d]);
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[j] = __builtin_fmaf(v[j], f, sum[j]);
            }
            if (d < dr) {
                if (whole) {
                    const float inv = L != 0.f ? 1.0f / L : 0.f;
                    const uint64_t at = (uint64_t)s * a.o_stride + (uint64_t)(h0 + h) * dr + d;
                    if (a.io_f16) {
                        half4_t r;
#pragma unroll
                        for (int j = 0; j < 4; ++j) r[j] = (_Float16)(sum[j] * inv);
                        *reinterpret_cast<half4_t*>(reinterpret_cast<_Float16*>(a.o) + at) = r;
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j) sum[j] *= inv;
                        *reinterpret_cast<float4_t*>(reinterpret_cast<float*>(a.o) + at) = sum;
                    }
                } else {
                    const uint64_t row = part * a.n_heads + h0 + h;
                    *reinterpret_cast<float4_t*>(a.scratch_out + row * dr + d) = sum;
                    if (d == 0u) { a.scratch_max[row] = M; a.scratch_sum[row] = L; }
                }
            }
        }
        __syncthreads();
    }
}

// Joins the parts of the sequences that lie in more than one workgroup's range: one workgroup per (head, sequence).  The parts are
// dealt to groups of D / 4 threads, each thread four columns.  Latency bound: 6.0 us for one sequence in 64 parts.
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedAttnLaunch a, uint32_t n_wg, uint32_t uk_shift) {
    __shared__ uint32_t red[2][kDecWaves];
    __shared__ float4_t sums[256];
    __shared__ float ls[256], ms[256];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const uint32_t head = blockIdx.x, s = blockIdx.y;
    const uint32_t mine = line_units(seq_units(a, paged_kv_len(a.s, s), uk_shift).units);
    uint32_t before = 0u, U = mine;
    if (a.s.n_seqs > 1u) {
        uint32_t all = 0u;
        for (uint32_t t = tid; t < a.s.n_seqs; t += 256u) {
            const uint32_t x = line_units(seq_units(a, paged_kv_len(a.s, t), uk_shift).units);
            all += x;
            before += t < s ? x : 0u;
        }
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) {
            before += __shfl_xor(before, off, kWave);
            all += __shfl_xor(all, off, kWave);
        }
        if (lane == 0) { red[0][w] = before; red[1][w] = all; }
        __syncthreads();
        before = red[0][0] + red[0][1] + red[0][2] + red[0][3];
        U = red[1][0] + red[1][1] + red[1][2] + red[1][3];
    }
    if (mine == 0u) return;
    // workgroup of unit u: the largest w with w U / N <= u
    n_wg = used_wgs(U, n_wg);
    const uint32_t wa = div_floor(((uint64_t)before + kBegin + 1u) * n_wg - 1u, U);   // of its first unit
    const uint32_t wb = div_floor(((uint64_t)before + mine) * n_wg - 1u, U);
    if (wa == wb) return;                                                // written by the workgroup itself
    const uint32_t dr = a.c.head_dim, quads = dr / 4u;
    const uint32_t groups = 256u / quads, grp = (uint32_t)tid / quads, q4 = (uint32_t)tid % quads;
    // (a range that begins inside the sequence, any but the first, has it as its first sequence)
    const uint32_t slot_a = div_floor((uint64_t)wa * U, n_wg) >= before ? 0u : 1u;
    auto part_row = [&](uint32_t x) { return ((uint64_t)x * 2u + (x == wa ? slot_a : 0u)) * a.n_heads + head; };
    // eight parts at a time, maxima, sums and outputs requested together: one trip to memory for up to 8 * groups parts
    constexpr int AT_ONCE = 8;
    float M = kNoScore, L = 0.f;
    float4_t sum = {0.f, 0.f, 0.f, 0.f};
    if (grp < groups) {
        for (uint32_t x0 = wa + grp; x0 <= wb; x0 += AT_ONCE * groups) {
            float m[AT_ONCE], l[AT_ONCE];
            float4_t v[AT_ONCE];
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                const uint32_t x = x0 + (uint32_t)i * groups;
                const uint64_t row = part_row(x <= wb ? x : wb);
                m[i] = a.scratch_max[row];
                l[i] = a.scratch_sum[row];
                v[i] = *reinterpret_cast<const float4_t*>(a.scratch_out + row * dr + q4 * 4u);
            }
            float mn = M;
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) mn = fmaxf(mn, m[i]);
            const float old = __builtin_amdgcn_exp2f(M - mn);
            M = mn;
            L *= old;
#pragma unroll
            for (int j = 0; j < 4; ++j) sum[j] *= old;
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                if (x0 + (uint32_t)i * groups > wb) break;
                const float f = __builtin_amdgcn_exp2f(m[i] - M);
                L = __builtin_fmaf(l[i], f, L);
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[j] = __builtin_fmaf(v[i][j], f, sum[j]);
            }
        }
    }
    sums[tid] = sum;
    ls[tid] = L;
    ms[tid] = M;
    __syncthreads();
    if (grp != 0u) return;
    float top = M;
    for (uint32_t x = 1; x < groups; ++x) top = fmaxf(top, ms[x * quads + q4]);
    const float own = __builtin_amdgcn_exp2f(M - top);
    L *= own;
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[j] *= own;
    for (uint32_t x = 1; x < groups; ++x) {
        const float4_t v = sums[x * quads + q4];
        const float f = __builtin_amdgcn_exp2f(ms[x * quads + q4] - top);
        L = __builtin_fmaf(ls[x * quads + q4], f, L);
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[j] = __builtin_fmaf(v[j], f, sum[j]);
    }
    const float inv = L != 0.f ? 1.0f / L : 0.f;
    const uint64_t at = (uint64_t)s * a.o_stride + (uint64_t)head * dr + q4 * 4u;
    if (a.io_f16) {
        half4_t r;
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = (_Float16)(sum[j] * inv);
        *reinterpret_cast<half4_t*>(reinterpret_cast<_Float16*>(a.o) + at) = r;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[j] *= inv;
        *reinterpret_cast<float4_t*>(reinterpret_cast<float*>(a.o) + at) = sum;
    }
}

uint32_t paged_decode_wgs(uint32_t head_groups) { return (512u + head_groups - 1u) / head_groups; }

namespace {

template <int DT, int D, int SUB>
hipError_t launch_dec(const PagedAttnLaunch& L, hipStream_t stream) {
    constexpr uint32_t UK = 16u * SUB;
    const uint32_t slices = (L.n_heads / L.c.n_kv_heads + kDecHeads - 1u) / kDecHeads;
    const uint32_t n_hg = L.c.n_kv_heads * slices;
    // an upper bound of the units from what the host knows
    uint64_t keys = L.max_kv;
    if (L.window != 0u && (uint64_t)L.window + L.n_sink + 2u * UK < keys) keys = (uint64_t)L.window + L.n_sink + 2u * UK;
    const uint64_t per_seq = (keys + UK - 1u) / UK;
    // A workgroup per sequence, without the prefix sums and without a join: up to eight units per wavefront, up to sixteen when there
    // are two workgroups per CU or more.  (FP8 heads of 128, 8 KV heads, dealt / a workgroup each: 64 sequences of 200-600 keys
    // 25.5 / 15.8 us, one of 1 000 12.8 / 11.8, 64 of 1 000-2 000 51.1 / 45.1, 16 of 1 000-4 000 25.4 / 32.1.)
    // (Rows of 512: a quarter of the wavefronts are resident and a unit is a longer way, so half of that, and from half a workgroup per
    // CU on.  64 FP8 sequences of 200-600 keys, 2 KV heads: 40.9 / 30.2 us; one of 1 000 22.5 / 37.3.)
    constexpr uint32_t SHORT = D == 512 ? 4u : 8u, FULL = D == 512 ? 128u : 512u;
    if (per_seq <= SHORT * kDecWaves || (per_seq <= 16u * kDecWaves && (uint64_t)L.s.n_seqs * n_hg >= FULL)) {
        hipLaunchKernelGGL((paged_decode_kernel<DT, D, SUB>), dim3(n_hg, L.s.n_seqs), dim3(256), 0, stream, L, L.s.n_seqs, slices, 1u);
        return hipGetLastError();
    }
    // as many workgroups as are resident: two per CU, one from rows of 256 on (FP8 rows of 256, 2 KV heads, 48 sequences of up to
    // 8 000 keys, two / one: 62.7 / 53.9 us; F32, 64 of 200-600: 54.5 / 40.3)
    uint64_t n = paged_decode_wgs(n_hg);
    if (D >= 256) n = (n + 1u) / 2u;
    const uint64_t useful = (L.s.n_seqs * (per_seq + kBegin) + kBegin + 2u * kDecWaves - 1u) / (kBegin + 2u * kDecWaves);
    if (n > useful) n = useful;
    const uint64_t fits = L.scratch_rows / (2u * (uint64_t)L.n_heads);
    if (n > fits) n = fits;
    if (n == 0u) n = 1u;
    hipLaunchKernelGGL((paged_decode_kernel<DT, D, SUB>), dim3(n_hg, (uint32_t)n), dim3(256), (L.s.n_seqs + 1u) * 4u, stream, L, (uint32_t)n, slices, 0u);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || n == 1u) return e;
    hipLaunchKernelGGL(paged_merge_kernel, dim3(L.n_heads, L.s.n_seqs), dim3(256), 0, stream, L, (uint32_t)n, (uint32_t)DecShape<DT, D, SUB>::SHIFT);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_paged_decode(const PagedAttnLaunch& L, hipStream_t stream) {
    const uint32_t d = L.c.head_dim;
    if (L.c.dtype == kF8) {
        if (d <= 64u) return launch_dec<kF8, 64, 4>(L, stream);
        if (d <= 128u) return launch_dec<kF8, 128, 2>(L, stream);
        if (d <= 256u) return launch_dec<kF8, 256, 2>(L, stream);
        return launch_dec<kF8, 512, 1>(L, stream);
    }
    if (L.c.dtype == kF16) {
        if (d <= 64u) return launch_dec<kF16, 64, 2>(L, stream);
        if (d <= 128u) return launch_dec<kF16, 128, 2>(L, stream);
        if (d <= 256u) return launch_dec<kF16, 256, 1>(L, stream);
        return launch_dec<kF16, 512, 1>(L, stream);
    }
    if (d <= 64u) return launch_dec<kF32, 64, 1>(L, stream);
    if (d <= 128u) return launch_dec<kF32, 128, 1>(L, stream);
    return launch_dec<kF32, 256, 1>(L, stream);
}

}  // namespace vfkv
