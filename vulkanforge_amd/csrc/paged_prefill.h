// Prefill attention over the paged cache: a ragged batch of chunks, causal, with a window per query and first tokens kept.
//
// o[r] = sum_j softmax_j(scale q[r].k_j) v_j over the keys row r sees; 4 * head_dim flop per visible (query row, key) pair, so
// for chunks of any length the matrix cores bound it.
//
//   - The query heads of one KV head and the tokens of a chunk form one line of rows (token major): a workgroup takes a block of
//     R = 32 NW consecutive rows of one sequence and one KV head, a wavefront 32 of them.  K and V are shared by the whole
//     group, and short chunks (drafted tokens) fill the tiles with heads.  Blocks are numbered by a prefix sum over the
//     batch that every workgroup forms itself (the offsets are device data), the last block of a sequence first: it has the most keys.
//   - Keys pass through LDS in tiles of KT, as f16 (or f32), once for all rows of the workgroup: global loads of tile t + 1 run
//     during the products of tile t, two LDS buffers, one barrier per tile.  A 16-key tile lies in one page, whose number is a
//     scalar load two tiles ahead.
//   - S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_32x32x16_f16: the scores of a row stay in one lane and its opposite half, P is
//     already where the second product wants it, V^T comes from the transposing LDS read.
//   - f16 queries enter as they are, f32 queries as f16 value + remainder, and the weights as value + remainder for both: f32-level
//     accuracy for one product more.  (Weights rounded to f16 are off by up to 2^-11 each, which large elements of V that cancel turn into
//     ten steps of an f16 output.)  F32 caches use the f32 matrix instruction.
//   - The running maximum is only raised when a score exceeds it by 2^8 (paged.h).
// Measured (f16 product of 8 192 x 8 192 matrices in the library: 1 175 TFLOP/s): 8 192 tokens from position 0, FP8, f16 rows,
// 32 / 8 / 128: 750-785 us by card = 700-735 TFLOP/s of useful work, 1 050-1 100 with the remainder product, the matrix units busy 0.50 and
// the vector units 0.45 of the time (LDS 0.25): the two wavefronts of a SIMD meet at the tile's barrier, so half of what could overlap
// does.  512 tokens over 4 096 keys, f32 rows: 83 us = 440 TFLOP/s of useful work, 880 with the remainder products.  Windows of 1 024
// keys, f16 rows: 507 (F16 pages) and 555 (FP8) TFLOP/s of useful work (18 tiles per block do not hide a block's beginning and end).  F32
// pages, 512 tokens over 4 096 keys: 328 us = 111 TFLOP/s of the f32 instruction's 154 in the library.  Tried and not kept: two row
// blocks per wavefront (one wavefront per SIMD, half the rate: the accumulators no longer fit the registers the matrix instructions
// take), tiles of 128 keys, raised wave priority around the products, the first tile requested before the queries (all within 3 %).
//
//   - Few rows over many keys: the tiles are cut into n_split parts over more workgroups and joined by paged_rows_merge_kernel.
#pragma once
#include <type_traits>

#include "device_utils.h"
#include "paged.h"

namespace vfkv {

namespace {

template <int DT, int D, int KT, int NW>
struct PreShape {
    static constexpr int ES = DT == kF32 ? 4 : DT == kF16 ? 2 : 1;
    static constexpr int LE = DT == kF32 ? 4 : 2;              // bytes per element in LDS
    static constexpr int CPR = D * ES / 16;                    // 16-byte chunks per cache row
    static constexpr int RPP = NW * 64 / CPR;                      // rows per staging pass
    static constexpr int NP = KT / RPP;                        // passes per tile and tensor
    // pitches: 16-byte reads of eight K rows, and reads of four (f16) / two (f32, four rows apart) V rows, hit distinct banks
    static constexpr int KPITCH = D * LE + 16;                 // bytes
    static constexpr int VPITCH = D * LE + (DT == kF32 ? 32 : 64);
    static constexpr int BUF = KT * (KPITCH + VPITCH);         // one buffer: K tile, V tile
    static_assert(KT % RPP == 0 || RPP > KT, "whole passes");
};

// Elements of a dword of the cache that are infinite or NaN, as a mask of their bits.
template <int DT>
__device__ __forceinline__ uint32_t not_finite(uint32_t x) {
    if constexpr (DT == kF32) return (x & 0x7F800000u) == 0x7F800000u ? 0xFFFFFFFFu : 0u;
    if constexpr (DT == kF16) return ((x & 0x7C00u) == 0x7C00u ? 0xFFFFu : 0u) | ((x & 0x7C000000u) == 0x7C000000u ? 0xFFFF0000u : 0u);
    const uint32_t top = ((x & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;        // E4M3FN: only codes 0x7F and 0xFF
    return top | (top - (top >> 7));
}

__device__ __forceinline__ float max_over_halves(float x) {
    float y = x;
    swap32(x, y);
    return fmaxf(x, y);
}

}  // namespace

// Exclusive prefix sums of the row blocks of the sequences, by the whole workgroup.
template <int NW>
__device__ __forceinline__ void block_prefix(const PagedAttnLaunch& a, uint32_t group, uint32_t rows, uint32_t* pre, uint32_t* wave_sum, int tid) {
    const int lane = tid & 63, w = tid >> 6;
    uint32_t carry = 0u;
    for (uint32_t base = 0; base < a.s.n_seqs; base += NW * 64u) {
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
        for (int i = 0; i < NW; ++i) {
            if (i < w) before += wave_sum[i];
            carry += wave_sum[i];
        }
        if (s < a.s.n_seqs) pre[s] = before + x - mine;
        __syncthreads();
    }
    if (tid == 0) pre[a.s.n_seqs] = carry;
    __syncthreads();
}

template <int DT, int D, bool IOF16, bool CAP, int KT, int CK, int NW, int MINW, int DS = 1>
__global__ __launch_bounds__(NW * 64, MINW) void paged_prefill_kernel(PagedAttnLaunch a, uint32_t n_split, uint32_t per_z) {
    using Z = PreShape<DT, D, KT, NW>;
    constexpr bool F32C = DT == kF32;
    constexpr bool QPAIR = !IOF16 && !F32C;                  // queries as value + remainder
    constexpr int NB = CK / 32;                              // 32-key blocks per chunk: what a wavefront takes through both products at once
    constexpr int DW = D / DS;                               // columns of a wavefront: DS wavefronts share 32 rows
    constexpr int DT32 = DW / 32;
    constexpr uint32_t R = 32u * NW / DS;
    static_assert(DS == 1 || (DS == 2 && KT == CK && !F32C), "the shared scores are joined once per tile");
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];   // two buffers; before the first tile, the prefix sums
    __shared__ uint32_t wave_sum[NW];
    // keys whose V row holds an infinity or NaN, from tiles that are hidden in part: at most the tiles the block's queries and
    // the two ends of its window cut through
    constexpr uint32_t kOddMax = KT * (2u * (R / KT + 2u) + 1u);
    __shared__ uint32_t n_odd, odd_key[kOddMax];
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n32 = lane & 31, hf = lane >> 5;
    // KV head fastest: consecutive workgroups go to different XCDs, so with eight heads each XCD keeps one head's keys in its L2
    const uint32_t group = a.n_heads / a.c.n_kv_heads, block_x = blockIdx.x / a.c.n_kv_heads, kvh = blockIdx.x - block_x * a.c.n_kv_heads;
    const uint32_t block = blockIdx.z * per_z + block_x;
    const uint32_t dr = a.c.head_dim;
    uint32_t* const pre = reinterpret_cast<uint32_t*>(lds);
    static_assert(2 * Z::BUF >= ((int)kPagedMaxSeqs + 1) * 4, "the prefix sums fit the tile buffers");
    if (tid == 0) n_odd = 0u;
    block_prefix<NW>(a, group, R, pre, wave_sum, tid);
    const uint32_t blocks = __builtin_amdgcn_readfirstlane(pre[a.s.n_seqs]);
    if (block >= blocks) return;
    const uint32_t bi = blocks - 1u - block;
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
    const uint32_t n_rows = (t1 - t0) * group;               // (n_tokens * n_heads <= 2^30)
    const uint32_t row0 = (bi - __builtin_amdgcn_readfirstlane(pre[s])) * R;
    if (row0 >= n_rows) return;                              // (offsets that overlap can wrap the sums of the line)
    __syncthreads();                                         // the prefix sums have been read: the buffers are free
    const uint32_t row1 = n_rows - row0 < R ? n_rows : row0 + R;
    const int kv_len = (int)__builtin_amdgcn_readfirstlane(paged_kv_len(a.s, s));
    const int pos0 = kv_len - (int)(t1 - t0);                // position of the chunk's first token
    const int pmin = pos0 + (int)(row0 / group), pmax = pos0 + (int)((row1 - 1u) / group);
    // key tiles of the block: first tokens in front of the window of its first query, then up to its last query, as far as there are rows
    auto keys_to = [&](int pos) { return pos < 0 ? 0u : (uint32_t)pos < a.s.limit ? (uint32_t)pos + 1u : a.s.limit; };
    const uint32_t n_keys = keys_to(pmax), all_see = keys_to(pmin);       // (every query sees up to all_see, its window aside)
    const uint32_t wlo = pmin > 0 ? paged_window_lo(a.window, (uint32_t)pmin) : 0u, lo_min = wlo < n_keys ? wlo : n_keys;
    const uint32_t first = lo_min / KT;
    const uint32_t sink = a.n_sink < lo_min ? a.n_sink : lo_min;
    const uint32_t su = (sink + KT - 1u) / KT;
    const uint32_t sink_tiles = su < first ? su : first;
    const uint32_t tiles = n_keys ? sink_tiles + (n_keys + KT - 1u) / KT - first : 0u;
    const uint32_t ta = (uint32_t)((uint64_t)blockIdx.y * tiles / n_split), tb = (uint32_t)((uint64_t)(blockIdx.y + 1u) * tiles / n_split);
    auto tile_key = [&](uint32_t t) { return (t < sink_tiles ? t : first + t - sink_tiles) * (uint32_t)KT; };

    // ---- this wavefront's rows
    const uint32_t wr0 = row0 + (uint32_t)(w / DS) * 32u, dw0 = (uint32_t)(w % DS) * DW;   // first row, first column
    const bool wave_has = wr0 < row1;
    const uint32_t wr1 = row1 < wr0 + 32u ? row1 : wr0 + 32u;
    const int wmin = wave_has ? pos0 + (int)(wr0 / group) : 0, wmax = wave_has ? pos0 + (int)((wr1 - 1u) / group) : -1;
    const int wave_sees = (int)keys_to(wmin);                // every query of the wavefront, its window aside
    const int wlo_max = wmax > 0 ? (int)paged_window_lo(a.window, (uint32_t)wmax) : 0;     // window start of the last query
    const int wlo_min = wmin > 0 ? (int)paged_window_lo(a.window, (uint32_t)wmin) : 0;
    uint32_t lo, span, lead;                     // a row sees the keys [lo, lo + span) and [0, lead)
    uint32_t tok, head;
    bool real;
    {
        const uint32_t r = wr0 + (uint32_t)n32;
        real = r < row1;
        const uint32_t rr = real ? r : row0;
        tok = rr / group;
        head = kvh * group + rr - tok * group;
        const int pos = real ? pos0 + (int)tok : -1;
        const uint32_t end = keys_to(pos);
        lo = pos > 0 ? paged_window_lo(a.window, (uint32_t)pos) : 0u;
        span = end > lo ? end - lo : 0u;
        lead = a.n_sink < end ? a.n_sink : end;
        tok += t0;
    }
    // ---- Q^T operands
    half8_t qh[F32C ? 1 : DW / 16], ql[QPAIR ? DW / 16 : 1];
    float qf[F32C ? D / 2 : 1];
    const float scale_l2 = a.scale * 1.44269504088896f;
    float qmul = scale_l2;                                   // of the scores, to log2 units
    {
        const uint64_t at = (uint64_t)tok * a.q_stride + (uint64_t)head * dr;
        if constexpr (F32C) {
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
                const uint32_t d = 8u * c + 4u * (uint32_t)hf;
                const bool ok = real && d < dr;
                float4_t x;
                if constexpr (IOF16) {
                    const half4_t h = *reinterpret_cast<const half4_t*>(reinterpret_cast<const _Float16*>(a.q) + at + (ok ? d : 0u));
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[j] = (float)h[j];
                } else {
                    x = *reinterpret_cast<const float4_t*>(reinterpret_cast<const float*>(a.q) + at + (ok ? d : 0u));
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) qf[4 * c + j] = ok ? x[j] : 0.f;
            }
        } else if constexpr (IOF16) {
#pragma unroll
            for (int c = 0; c < DW / 16; ++c) {
                const uint32_t d = dw0 + 16u * c + 8u * (uint32_t)hf;
                const bool ok = real && d < dr;
                const half8_t x = *reinterpret_cast<const half8_t*>(reinterpret_cast<const _Float16*>(a.q) + at + (ok ? d : 0u));
#pragma unroll
                for (int j = 0; j < 8; ++j) qh[c][j] = ok ? x[j] : (_Float16)0.f;
            }
        } else {
            // times the power of two that brings the row's largest element to [0.5, 1): value + remainder hold every element to 2^-23 of
            // that, whatever the row's size
            float x[DW / 16][8], top = 0.f;
#pragma unroll
            for (int c = 0; c < DW / 16; ++c) {
                const uint32_t d = dw0 + 16u * c + 8u * (uint32_t)hf;
                const bool ok = real && d < dr;
                const float* const src = reinterpret_cast<const float*>(a.q) + at + (ok ? d : 0u);
                const float4_t x0 = *reinterpret_cast<const float4_t*>(src), x1 = *reinterpret_cast<const float4_t*>(src + 4);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    x[c][j] = ok ? (j < 4 ? x0[j & 3] : x1[j & 3]) : 0.f;
                    top = fmaxf(top, fabsf(x[c][j]));
                }
            }
            top = max_over_halves(top);
            if constexpr (DS > 1) {                          // the other wavefront's columns of the same rows
                float* const tops = reinterpret_cast<float*>(lds + 2 * Z::BUF);
                tops[w * 64 + lane] = top;
                __syncthreads();
                top = fmaxf(top, tops[(w ^ 1) * 64 + lane]);
            }
            const int e = __builtin_amdgcn_frexp_expf(top);
            qmul = fmaxf(__builtin_ldexpf(scale_l2, e), 1e-37f);   // (not 0: -inf * 0 of a hidden key would be NaN)
#pragma unroll
            for (int c = 0; c < DW / 16; ++c)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float y = __builtin_ldexpf(x[c][j], -e);
                    const _Float16 hi = (_Float16)y;
                    qh[c][j] = hi;
                    ql[c][j] = (_Float16)(y - (float)hi);
                }
        }
    }

    float16_t acc[DT32];
    float m = kNoScore, l = 0.f;                             // l: this lane's keys only, summed at the end
    uint32_t far = 0u;                                       // some row is far out: its products are rounded before they are compared
#pragma unroll
    for (int n = 0; n < DT32; ++n)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[n][e] = 0.f;
    const float cap_l2 = a.softcap * 1.44269504088896f;
    const float inv_cap_l2 = CAP ? 1.0f / cap_l2 : 0.f;
    const float fac = CAP ? 1.0f : qmul;                 // scores are kept unscaled; the soft-cap leaves them in log2 units

    // ---- staging
    const uint32_t row_b = dr * Z::ES;
    const uint32_t chunk = (uint32_t)tid % Z::CPR, srow = (uint32_t)tid / Z::CPR;
    const bool chunk_ok = chunk * 16u < row_b;
    const uint64_t head_rows = (uint64_t)kvh << a.c.page_shift;
    const uint32_t slot_mask = (1u << a.c.page_shift) - 1u;
    const int32_t* const table = a.s.table + (uint64_t)s * a.s.table_stride;
    constexpr int NP = Z::NP < 1 ? 1 : Z::NP;
    constexpr int SUBS = KT / 16;                            // 16-key tiles: each lies in one page
    struct Pages {
        uint32_t tile[SUBS];                                 // pages of the tile, for masking
        uint32_t pass[NP];                                   // pages of the rows this wavefront stages (one page per wavefront and pass)
    };
    const uint32_t wave_row = (uint32_t)w * (64u / Z::CPR);
    auto page_at = [&](uint32_t key) { return (uint32_t)table[(key < n_keys ? key : n_keys - 1u) >> a.c.page_shift]; };
    auto get_pages = [&](uint32_t t) {
        Pages r;
        const uint32_t kb = tile_key(t < tb ? t : tb - 1u);
#pragma unroll
        for (int i = 0; i < SUBS; ++i) r.tile[i] = page_at(kb + 16u * i);
#pragma unroll
        for (int p = 0; p < NP; ++p) r.pass[p] = page_at(kb + (((uint32_t)(p * Z::RPP) + wave_row) & (KT - 16u)));
        return r;
    };
    u32x4 kraw[NP], vraw[NP];
    auto fetch = [&](const Pages& P, uint32_t t) {
        const uint32_t kb = tile_key(t);
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            const uint32_t page = P.pass[p] < a.c.n_pages ? P.pass[p] : 0u;
            const uint32_t key = kb + (((uint32_t)(p * Z::RPP) + wave_row) & (KT - 16u));
            const uint64_t off = (uint64_t)page * a.c.page_bytes + (head_rows + (key & slot_mask)) * row_b;
            const uint32_t lane_off = (((uint32_t)(p * Z::RPP) + srow) & 15u) * row_b + (chunk_ok ? chunk * 16u : 0u);
            kraw[p] = *reinterpret_cast<const u32x4*>(a.c.k + off + lane_off);
            vraw[p] = *reinterpret_cast<const u32x4*>(a.c.v + off + lane_off);
        }
    };
    // In a tile that some query of the block does not see completely, V rows no query sees become zeros (their weights are zero, but
    // 0 * NaN of a stale row is not), and so does every element that is not finite: queries the key is hidden from
    // must not meet it.  The key is noted and the queries that do see it get the element when the output is written.
    auto stage = [&](int buf, const Pages& P, uint32_t t) {
        uint8_t* const kl = lds + buf * Z::BUF;
        uint8_t* const vl = kl + KT * Z::KPITCH;
        const uint32_t kb = tile_key(t);
        const bool hidden = kb + KT > all_see ||
                            !(kb + KT <= a.n_sink || a.window == 0u || kb >= paged_window_lo(a.window, (uint32_t)pmax));
        bool part = hidden;
#pragma unroll
        for (int i = 0; i < SUBS; ++i) part = part || P.tile[i] >= a.c.n_pages;
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            const uint32_t row = (uint32_t)(p * Z::RPP) + srow;
            u32x4 k = kraw[p], v = vraw[p];
            if (part) {
                const uint32_t key = kb + row;
                const bool ok = chunk_ok && key < n_keys && (key >= lo_min || key < sink) && P.pass[p] < a.c.n_pages;
                bool odd = false;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t bad = not_finite<DT>(v[i]);
                    odd = odd || (ok && bad != 0u);
                    v[i] = ok ? (hidden ? v[i] & ~bad : v[i]) : 0u;
                }
                if (hidden && odd && row < (uint32_t)KT) {
                    const uint64_t same = __ballot(odd) >> ((uint32_t)lane / Z::CPR * Z::CPR);   // (this lane's row: CPR lanes from there)
                    if ((uint32_t)__builtin_ctzll(same) == (uint32_t)lane % Z::CPR) {
                        const uint32_t at = atomicAdd(&n_odd, 1u);
                        if (at < kOddMax) odd_key[at] = key;
                    }
                }
            }
            if (!chunk_ok || (Z::RPP > KT && row >= (uint32_t)KT)) continue;      // (columns past a narrower head stay zero)
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
    };

    // ---- one tile
    auto scores = [&](float16_t (&sc)[NB], int buf, int chunk_at) {
        const uint8_t* const kl = lds + buf * Z::BUF + chunk_at * Z::KPITCH + dw0 * Z::LE;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int e = 0; e < 16; ++e) sc[b][e] = 0.f;
            const uint8_t* const krow = kl + (32 * b + n32) * Z::KPITCH + hf * 16;
            if constexpr (F32C) {
#pragma unroll
                for (int c = 0; c < D / 8; ++c) {
                    const float4_t k = *reinterpret_cast<const float4_t*>(krow + 32 * c);
#pragma unroll
                    for (int j = 0; j < 4; ++j) sc[b] = __builtin_amdgcn_mfma_f32_32x32x2f32(k[j], qf[4 * c + j], sc[b], 0, 0, 0);
                }
            } else {
#pragma unroll
                for (int c = 0; c < DW / 16; ++c) {
                    const half8_t k = *reinterpret_cast<const half8_t*>(krow + 32 * c);
                    sc[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qh[c], sc[b], 0, 0, 0);
                    if constexpr (QPAIR) sc[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, ql[c], sc[b], 0, 0, 0);
                }
            }
        }
    };
    auto finish = [&](float16_t (&sc)[NB], bool masked, int buf, const uint32_t (&pages)[CK / 16], int chunk_at, int kb) {   // masked: some of the queries do not see some of the keys
        const uint8_t* const vl = lds + buf * Z::BUF + KT * Z::KPITCH + chunk_at * Z::VPITCH + dw0 * Z::LE;
        if constexpr (CAP) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int e = 0; e < 16; ++e) sc[b][e] = paged_softcap_l2(sc[b][e] * qmul, cap_l2, inv_cap_l2);
        }
        float f = fac;
        bool rounded = false;
        auto round_products = [&](bool mine) {               // of this lane's row; the others keep theirs
            const float by = mine ? fac : 1.0f;
            f = mine ? 1.0f : f;
            rounded = rounded || mine;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int e = 0; e < 16; ++e) sc[b][e] *= by;
        };
        if (!CAP && __builtin_expect(far != 0u, 0)) round_products(paged_far(m));
        if (masked) {
            // key in [lo, pos] as one unsigned comparison against their number; a key among the first tokens as another
            auto hide = [&](auto firsts) {
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const bool there = pages[2 * b + h] < a.c.n_pages;      // (uniform: 16 keys lie in one page)
                        const uint32_t key = (uint32_t)(kb + 32 * b + 16 * h + 4 * hf), rel = key - lo;
                        const uint32_t some = there ? span : 0u, front = there ? lead : 0u;
#pragma unroll
                        for (uint32_t x = 0; x < 8; ++x) {
                            const uint32_t off = 8u * (x / 4u) + x % 4u;
                            bool seen = rel + off < some;
                            if constexpr (decltype(firsts)::value) seen = seen || key + off < front;
                            sc[b][8 * h + x] = seen ? sc[b][8 * h + x] : -__builtin_inff();
                        }
                    }
            };
            if ((uint32_t)kb < a.n_sink) hide(std::true_type{}); else hide(std::false_type{});
        }
        float mx = sc[0][0];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) mx = fmaxf(mx, sc[b][e]);
        if (__any(mx * f - m > kRaise + kBias<DT>)) {
            const float mn = fmaxf(m, max_over_halves(mx * f) - kBias<DT>);
            if constexpr (!CAP) {
                far = __builtin_amdgcn_readfirstlane(__any(paged_far(mn)) ? 1u : 0u);
                if (__builtin_expect(far != 0u, 0)) round_products(paged_far(mn) && !rounded);
            }
            const float corr = __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= corr;
#pragma unroll
            for (int n = 0; n < DT32; ++n)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[n][e] *= corr;
        }
        float sum = 0.f;                                     // of the chunk first: one by one, small weights would not reach a large l
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                sc[b][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[b][e], f, -m));
                sum += sc[b][e];
            }
        l += sum;
        if constexpr (F32C) {
            // (the instruction adds two keys at a time: the chunk's sum first, for the same reason)
#pragma unroll
            for (int n = 0; n < DT32; ++n) {
                float16_t part;
#pragma unroll
                for (int e = 0; e < 16; ++e) part[e] = 0.f;
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float v = *reinterpret_cast<const float*>(vl + (32 * b + 8 * (e / 4) + 4 * hf + e % 4) * Z::VPITCH + n32 * 4 + 128 * n);
                        part = __builtin_amdgcn_mfma_f32_32x32x2f32(v, sc[b][e], part, 0, 0, 0);
                    }
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[n][e] += part[e];
                // (the next columns' loads, moved up to here, spill: 512 x 4 608, rows of 128, 356 us against 328)
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
            // lane's place in the transposing read: row 4 hf + (lane % 16) / 4 of eight-row steps, column group of its sixteen lanes
            const uint8_t* const vlane = vl + (4 * hf + (lane & 15) / 4) * Z::VPITCH + (16 * ((lane >> 4) & 1) + 4 * (lane & 3)) * 2;
#pragma unroll
            for (int kk = 0; kk < CK / 16; ++kk) {
                uint32_t h[4], r[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p0 = sc[kk / 2][8 * (kk % 2) + 2 * i], p1 = sc[kk / 2][8 * (kk % 2) + 2 * i + 1];
                    h[i] = __builtin_bit_cast(uint32_t, half2_t{(_Float16)p0, (_Float16)p1});
                    r[i] = pack_f16_remainder(p0, p1, h[i]);
                }
                const half8_t ph = __builtin_bit_cast(half8_t, h), pl = __builtin_bit_cast(half8_t, r);
#pragma unroll
                for (int n = 0; n < DT32; ++n) {
                    const half4_t v0 = lds_read_tr16(reinterpret_cast<const _Float16*>(vlane + 16 * kk * Z::VPITCH + 64 * n));
                    const half4_t v1 = lds_read_tr16(reinterpret_cast<const _Float16*>(vlane + (16 * kk + 8) * Z::VPITCH + 64 * n));
                    const half8_t v = __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
                    acc[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, ph, acc[n], 0, 0, 0);
                    acc[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pl, acc[n], 0, 0, 0);
                }
            }
        }
    };

    if (dr < (uint32_t)D)                                    // columns past a narrower head: zeros in both buffers, for good
        for (uint32_t i = (uint32_t)tid * 16u; i < 2u * Z::BUF; i += NW * 1024u) *reinterpret_cast<u32x4*>(lds + i) = u32x4{0u, 0u, 0u, 0u};
    if (ta < tb) {
        if (dr < (uint32_t)D) __syncthreads();
        Pages p0 = get_pages(ta), p1 = get_pages(ta + 1u);
        fetch(p0, ta);
        stage(0, p0, ta);
        for (uint32_t t = ta; t < tb; ++t) {
            const int buf = (int)((t - ta) & 1u);
            __syncthreads();                                   // tile t staged by all; tile t - 1 no longer read
            const Pages p2 = get_pages(t + 2u);
            if (t + 1u < tb) fetch(p1, t + 1u);
            if (wave_has || DS > 1) {
                auto one = [&](int c) {
                    const int kb = (int)tile_key(t) + c;
                    uint32_t pages[CK / 16];
                    bool ghost = false;
#pragma unroll
                    for (int i = 0; i < CK / 16; ++i) {
                        pages[i] = p0.tile[i];
#pragma unroll
                        for (int x = 1; x < KT / CK; ++x) pages[i] = c == x * CK ? p0.tile[x * (CK / 16) + i] : pages[i];
                        ghost = ghost || pages[i] >= a.c.n_pages;
                    }
                    // (a chunk that none of the wavefront's queries sees is passed over)
                    const bool none = kb > wmax || ((uint32_t)kb >= a.n_sink && kb + CK <= wlo_min);
                    auto masked = [&] { return !(kb + CK <= wave_sees && (kb >= wlo_max || (uint32_t)(kb + CK) <= a.n_sink) && !ghost); };
                    if constexpr (DS == 1) {
                        if (none) return;
                        float16_t sc[NB];
                        scores(sc, buf, c);
                        finish(sc, masked(), buf, pages, c, kb);
                    } else {                                    // sums over half of the columns each: added, in either order the same
                        float4_t* const mine = reinterpret_cast<float4_t*>(lds + 2 * Z::BUF) + w * (NB * 256) + lane;
                        const float4_t* const other = reinterpret_cast<const float4_t*>(lds + 2 * Z::BUF) + (w ^ 1) * (NB * 256) + lane;
                        float16_t sc[NB];
                        const bool any = wave_has && !none;
                        if (any) {
                            scores(sc, buf, c);
#pragma unroll
                            for (int x = 0; x < 4 * NB; ++x)
                                mine[64 * x] = float4_t{sc[x / 4][4 * (x % 4)], sc[x / 4][4 * (x % 4) + 1], sc[x / 4][4 * (x % 4) + 2], sc[x / 4][4 * (x % 4) + 3]};
                        }
                        __syncthreads();
                        if (any) {
#pragma unroll
                            for (int x = 0; x < 4 * NB; ++x) {
                                const float4_t y = other[64 * x];
#pragma unroll
                                for (int j = 0; j < 4; ++j) sc[x / 4][4 * (x % 4) + j] += y[j];
                            }
                            finish(sc, masked(), buf, pages, c, kb);
                        }
                    }
                };
                if constexpr (KT == CK) one(0);
                else
#pragma unroll 1
                    for (int c = 0; c < KT; c += CK) one(c);
            }
            if (t + 1u < tb) stage(buf ^ 1, p1, t + 1u);
            p0 = p1;
            p1 = p2;
        }
    }

    // ---- output
    const float L = xor32_sum(l);
    const uint64_t row = ((uint64_t)tok * a.n_heads + head) * n_split + blockIdx.y;
    const uint64_t at = (uint64_t)tok * a.o_stride + (uint64_t)head * dr;
    if (real) {
        const float inv = n_split > 1u ? 1.0f : L != 0.f ? 1.0f / L : 0.f;
        if (n_split > 1u && hf == 0 && dw0 == 0u) { a.scratch_max[row] = m; a.scratch_sum[row] = L; }
#pragma unroll
        for (int n = 0; n < DT32; ++n)
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const uint32_t d = dw0 + 32u * n + 8u * b + 4u * (uint32_t)hf;
                if (d >= dr) continue;
                float4_t v;
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = acc[n][4 * b + j] * inv;
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
    // ---- noted keys: their infinities and NaNs go to the rows that see them, each lane on the elements it has just written
    if (ta >= tb) return;
    __syncthreads();                                         // the last tile's notes
    const uint32_t n_bad = __builtin_amdgcn_readfirstlane(n_odd < kOddMax ? n_odd : kOddMax);
#pragma unroll 1
    for (uint32_t i = 0; i < n_bad; ++i) {
        const uint32_t key = __builtin_amdgcn_readfirstlane(odd_key[i]);
        const uint32_t page = (uint32_t)table[key >> a.c.page_shift];
        const uint8_t* const vrow = a.c.v + (uint64_t)(page < a.c.n_pages ? page : 0u) * a.c.page_bytes + (head_rows + (key & slot_mask)) * row_b;
        if (!real || !(key - lo < span || key < lead)) continue;
#pragma unroll 1
        for (uint32_t d = dw0 + 4u * (uint32_t)hf; d < dr && d < dw0 + DW; d += 8u)
#pragma unroll 1
            for (uint32_t j = d; j < d + 4u; ++j) {
                const float v = load_kv_elem(vrow, DT, j);
                if (fabsf(v) < __builtin_inff()) continue;
                if (n_split > 1u) a.scratch_out[row * dr + j] += v;
                else if constexpr (IOF16) reinterpret_cast<_Float16*>(a.o)[at + j] = (_Float16)((float)reinterpret_cast<_Float16*>(a.o)[at + j] + v);
                else reinterpret_cast<float*>(a.o)[at + j] += v;
            }
    }
}

namespace {

// Whether the blocks of a chunk see about as many keys each: a context in front of it, or a window that is short against it.
bool blocks_alike(const PagedAttnLaunch& L) {
    const uint64_t chunk = (L.s.n_tokens + L.s.n_seqs - 1u) / L.s.n_seqs;
    return L.max_kv >= 2u * chunk || (L.window != 0u && chunk >= 2u * (uint64_t)L.window);
}

template <int DT, int D, bool IOF16, bool CAP, int KT, int CK, int NW, int MINW, int DS = 1>
hipError_t launch_pre(const PagedAttnLaunch& L, hipStream_t stream) {
    using Z = PreShape<DT, D, KT, NW>;
    constexpr uint64_t R = 32u * NW / DS;
    constexpr uint32_t LDS = 2u * Z::BUF + (DS > 1 ? NW * 64u * CK * 2u : 0u);   // (DS > 1: the scores in f32)
    const uint64_t group = L.n_heads / L.c.n_kv_heads;
    // a sequence's last block may be ragged: at most one block more per sequence that has rows
    const uint64_t with_rows = L.s.n_seqs < L.s.n_tokens ? L.s.n_seqs : L.s.n_tokens;
    uint64_t blocks = L.s.n_tokens * group / R + with_rows;
    if (blocks > L.s.n_tokens * group) blocks = L.s.n_tokens * group;
    // a dimension of a launch holds fewer than 2^32 threads: the rest of the blocks along z (at most 2^30 workgroups in all)
    const uint64_t room_x = 0xFFFFFFFFull / (NW * 64u) / L.c.n_kv_heads, per_z = blocks < room_x ? blocks : room_x;
    if (per_z == 0u || (blocks + per_z - 1u) / per_z > 65535u) return hipErrorInvalidValue;   // (not with n_tokens * n_heads <= 2^30)
    // Split over the keys, as long as the card has room and a part has a tile: the tiles of a part against the join, which writes and
    // reads the parts once (about 4 TB/s and 3 us).  A tile takes 1.8 us (four wavefronts) to 2.5 us (eight) for f16 rows of 128
    // elements, 1.6 times that for f32 rows, 6.8 us for 32 keys on the f32 instruction.  (FP8, 32 / 8 / 128, one part against two: 1 024
    // f16 tokens from position 0 38.1 / 45.9 us, over 5 000 keys 237 / 150 us; 7 tokens over 1 000 keys, F16 heads of 64, 4 / 16 parts
    // 15.0 / 11.3 us.)
    constexpr uint64_t tile_ns = (DT == kF32 ? 6800u * KT / 32u : (IOF16 ? 2200u : 3500u) * KT / 64u) * (D / DS) / 128u;
    const uint64_t likely = (L.s.n_tokens * group + R - 1u) / R * L.c.n_kv_heads;
    // (unlike blocks: twice the workgroups that fit, so that the last ones are short; F16 rows of 256, 2 048 tokens 129 -> 105 us)
    const uint64_t room = 256u * MINW * 4u / NW * (blocks_alike(L) ? 1u : 2u);
    uint64_t keys = L.max_kv;
    if (L.window != 0u && (uint64_t)L.window + L.n_sink + R + 2u * KT < keys) keys = (uint64_t)L.window + L.n_sink + R + 2u * KT;
    const uint64_t tiles = (keys + KT - 1u) / KT, rows = (uint64_t)L.s.n_tokens * L.n_heads;
    uint64_t most = room / likely;
    if (most > tiles) most = tiles;
    if (most > L.scratch_rows / rows) most = L.scratch_rows / rows;
    if (most > 64u) most = 64u;
    uint64_t n = 1u, best = tiles * tile_ns;
    for (uint64_t i = 2u; i <= most; ++i) {
        const uint64_t ns = (tiles + i - 1u) / i * tile_ns + 3000u + rows * i * L.c.head_dim * 8u / 4000u;
        if (ns < best) { best = ns; n = i; }
    }
    hipLaunchKernelGGL((paged_prefill_kernel<DT, D, IOF16, CAP, KT, CK, NW, MINW, DS>), dim3((uint32_t)(per_z * L.c.n_kv_heads), (uint32_t)n, (uint32_t)((blocks + per_z - 1u) / per_z)),
                       dim3(NW * 64), LDS, stream, L, (uint32_t)n, (uint32_t)per_z);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || n == 1u) return e;
    return launch_paged_rows_merge(L, (uint32_t)n, stream);
}

template <int DT, bool IOF16, bool CAP>
hipError_t launch_dim(const PagedAttnLaunch& L, hipStream_t stream) {
    const uint32_t d = L.c.head_dim;
    if constexpr (DT == kF32) {
        if (d <= 64u) return launch_pre<DT, 64, IOF16, CAP, 32, 32, 4, 2>(L, stream);
        if (d <= 128u) return launch_pre<DT, 128, IOF16, CAP, 32, 32, 4, 2>(L, stream);
        return launch_pre<DT, 256, IOF16, CAP, 32, 32, 4, 1>(L, stream);
    } else {
        // Workgroups of eight wavefronts share a staged tile among twice the rows, but a card that they fill only once waits for the
        // block with the most keys: they are taken for chunks that fill blocks of 256 rows, with two rounds of blocks or with a
        // context that makes the blocks alike.  (FP8 / f16 rows of 128, eight / four wavefronts: 4 096 tokens from position 0
        // 203 / 222 us, 2 048 90 / 76 us, 1 024 tokens over 5 000 keys 150 / 159 us; F16 rows of 256: 8 192 tokens 953 / 1 204 us,
        // 4 096 424 / 323 us, 2 048 over 6 000 keys 476 / 571 us.  At 256 elements the eight spill 20 (FP8) or 34 (F16) registers, counted
        // in these figures.)
        const uint64_t rows = (uint64_t)L.s.n_tokens * (L.n_heads / L.c.n_kv_heads);
        // Short windows, rows of up to 128: two workgroups of four on a CU, one of which begins or ends a block while the other
        // computes.  (Eight / four: FP8 / f16 rows, 2 x 4 096 tokens, window 128 102 / 86 us, 4 096, window 512 84 / 78, 8 192, window 1 024 250 / 232,
        // 4 096 over 16 384, window 4 096 392 / 403; F16 pages 107 / 97, 86.3 / 85.7, 259 / 255, 411 / 442; FP8 / f32 rows 109 / 99,
        // 90 / 92, 289 / 280, 479 / 500.  Between 384 and 1 536 the two are within 2 % over F16 pages and within 3 % for f32 rows.)
        const bool brief = d <= 128u && L.window != 0u && (uint64_t)L.window + L.n_sink <= (DT == kF8 && IOF16 ? 1536u : 384u);
        const bool many = !brief && rows >= 256ull * L.s.n_seqs && (blocks_alike(L) || rows / 256u * L.c.n_kv_heads >= 512u);
        constexpr int CK = IOF16 ? 64 : 32, KT = 64;
        if (d <= 64u) return many ? launch_pre<DT, 64, IOF16, CAP, 64, 64, 8, 2>(L, stream) : launch_pre<DT, 64, IOF16, CAP, 64, 64, 4, 2>(L, stream);
        if (d <= 128u) return many ? launch_pre<DT, 128, IOF16, CAP, KT, CK, 8, 2>(L, stream) : launch_pre<DT, 128, IOF16, CAP, KT, CK, 4, 2>(L, stream);
        // rows of 512: two wavefronts per block of 32 rows, each half of the columns of both products, their scores added through LDS
        // (16 / 2 heads, FP8, f16 rows: 512 tokens over 4 096 keys 219 us = 333 TFLOP/s of useful work, 4 096 from position 0 755 us = 364;
        // one workgroup per CU, two barriers per tile; the generic kernel: 43 ms)
        if (d > 256u) return launch_pre<DT, 512, IOF16, CAP, 32, 32, 4, 1, 2>(L, stream);
        if constexpr (IOF16)                                     // (value + remainder of 256 elements do not fit 256 registers)
            if (many) return launch_pre<DT, 256, IOF16, CAP, 32, 32, 8, 2>(L, stream);
        return launch_pre<DT, 256, IOF16, CAP, 32, 32, 4, 1>(L, stream);
    }
}

}  // namespace

// One translation unit per cache type: paged_prefill_{full,half,byte}.hip.
template <int DT>
hipError_t launch_prefill_of(const PagedAttnLaunch& L, hipStream_t stream) {
    if (L.softcap > 0.f) return L.io_f16 ? launch_dim<DT, true, true>(L, stream) : launch_dim<DT, false, true>(L, stream);
    return L.io_f16 ? launch_dim<DT, true, false>(L, stream) : launch_dim<DT, false, false>(L, stream);
}

}  // namespace vfkv
