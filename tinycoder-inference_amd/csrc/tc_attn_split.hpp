// tc_attn_split.hpp -- attention of up to 16 rows per key/value head: decode steps and
// a few drafted tokens. HBM-bound: every cached key and value of a head is read once
// for all its rows.
//
// The line of tiles (32 tokens for 16 rows) is cut into equal parts, one per
// workgroup. The waves of a workgroup take its tiles in turn, each through LDS of its
// own and without barriers: keys of the next tile are on their way while the values
// of this one are multiplied, and the other way round. Where a sequence's tiles end or
// the part does, the waves join their sums. Rows whose tiles lie in several parts
// leave unnormalised sums, which k_attn_join adds up.
#pragma once

#include "tc_attn_kernel.hpp"

namespace tc {
namespace {

// Shape of a launch for one cache type, number of pieces and padded head size.
template <int CT, int NP, int DP>
struct SplitShape {
    static constexpr int R = 16, NW = 4, STRETCH = 128;
    static constexpr int ES = scaled_type(CT) ? 1 : 2;
    static constexpr int RB = DP * ES;                        // bytes of a cache row in LDS
    static constexpr int TILE = kTileTokens * RB;             // of a tile of keys or values
    static constexpr int SCALES = scaled_type(CT) ? 768 : 0;  // factors, two tiles'; log2 and reciprocal
    static constexpr int WAVE = 2 * TILE + SCALES;
    static constexpr int MISC = 6144;  // (the first bytes of LDS hold the small things)
    static constexpr int LDS = MISC + NW * WAVE;
    // workgroups per CU: what LDS allows, up to 4 (128 registers a lane)
    static constexpr int BY_LDS = 160 * 1024 / LDS;
    static constexpr int BY_REG = DP == 256 || NP == 3 ? 2 : 3;
    static constexpr int OCC = BY_LDS < BY_REG ? BY_LDS : BY_REG;
};

struct SplitMisc {
    float m[4][16], l[4][16], inv[16];
    LineMisc line;
    RunMisc<128> runs;
};
static_assert(sizeof(SplitMisc) <= 6144, "");

template <int CT, int NP, int DP>
__global__ __launch_bounds__((64 * SplitShape<CT, NP, DP>::NW), (SplitShape<CT, NP, DP>::OCC)) void k_attn_split(
    AttnArgs a, RowRange rg, SplitScratch sc) {
    using Sh = SplitShape<CT, NP, DP>;
    constexpr int R = Sh::R, ES = Sh::ES, RB = Sh::RB, NW = Sh::NW;
    using Ge = Geo<R, DP>;
    constexpr int KS = Ge::KS, DB = Ge::DB, NS = Ge::NS;
    constexpr bool SCALED = scaled_type(CT);
    extern __shared__ __align__(1024) unsigned char lds[];
    SplitMisc &ms = *reinterpret_cast<SplitMisc *>(lds);
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t col = lane % R, g = lane / R;
    unsigned char *const mine = lds + Sh::MISC + wave * Sh::WAVE;
    const uint32_t ktile = lds_addr(lds) + Sh::MISC + wave * Sh::WAVE, vtile = ktile + Sh::TILE;
    float *const raw = reinterpret_cast<float *>(mine + 2 * Sh::TILE);  // [2][64] a tile's factors: keys', values'
    float *const lv = raw + 128, *const iv = raw + 160;                 // [32] log2 and reciprocal of the values'
    const uint32_t D = a.kv.dim, rowbytes = D * ES, run_bytes = 16 * rowbytes, nch = rowbytes / 16;

    uint64_t part, left;
    Place pl = line_part<R, kTileTokens, 64 * NW>(a, rg, blockIdx.x, gridDim.x, NW, ms.line, tid, &part, &left);
    if (tid == 0) sc.jobs[blockIdx.x].count = 0;

    bool first_seg = true;
    while (left != 0) {
        const uint32_t seq = pl.seq, r0 = pl.r0, kvh = pl.kvh, off = pl.off;
        const RowBlock b = row_block<R, kTileTokens>(a, seq, r0);
        const uint32_t seg = uint32_t(min(uint64_t(b.tiles - off), left));

        const uint32_t row = r0 + col;
        u32x4 q[NP][KS];
        const float factor = load_q<CT, NP, R, DP, ES>(a, b.begin, kvh, row, b.rows, g, q);
        const int32_t pos = row < b.rows ? b.pos0 + int32_t(row / a.group) : -1;  // the lane's row sees tokens up to here
        const int32_t from = a.window != 0 && int64_t(pos) + 1 > int64_t(a.window) ? int32_t(pos + 1 - a.window) : 0;

        constexpr int LPR = RB / 16, RPI = 64 / LPR;  // lanes per row, rows per load
        constexpr int LOADS = 2 * (16 / RPI);         // loads of a tile of keys or values
        auto load = [&](uint32_t dst, const uint8_t *src, const TileRuns &w, auto swizzle) __attribute__((always_inline)) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint8_t *at = src + uint64_t(w.run[h]) * run_bytes;
#pragma unroll
                for (int j = 0; j < 16 / RPI; ++j) {
                    const uint32_t r = j * RPI + lane / LPR, c = (lane % LPR) ^ swizzle(16 * h + r);
                    // (dims past the row's: others of it, which meet zeros of q, or go nowhere)
                    dma16(dst + (16 * h + j * RPI) * RB, at, r * rowbytes + (c < nch ? 16 * c : 0));
                }
            }
        };
        auto load_k = [&](const TileRuns &w) __attribute__((always_inline)) { load(ktile, a.kv.k, w, key_swizzle<R, RB>); };
        auto load_v = [&](const TileRuns &w) __attribute__((always_inline)) { load(vtile, a.kv.v, w, value_swizzle<R, RB, ES>); };
        // lanes 0-31 the keys' factors of the 32 tokens, the others the values'
        auto load_scales = [&](const TileRuns &w, uint32_t odd) __attribute__((always_inline)) {
            const float *p = lane >= 32 ? a.kv.vs : a.kv.ks;
            dma4(ktile + 2 * Sh::TILE + 256 * odd, p + 16 * uint64_t(lane & 16 ? w.run[1] : w.run[0]) + (lane & 15));
        };

        Acc<R> o[DB];
#pragma unroll
        for (int d = 0; d < DB; ++d) o[d] = Acc<R>{};
        float m = kNegInf, l = 0.0f;

        for (uint32_t c0 = off; c0 < off + seg; c0 += Sh::STRETCH) {
            const uint32_t t_end = min(off + seg, c0 + Sh::STRETCH);
            __syncthreads();
            find_runs<64 * NW>(a, seq, kvh, b.lo + 32 * int32_t(c0), b.hi, t_end - c0, ms.runs, tid);
            __syncthreads();
            uint32_t t = c0 + wave;
            uint32_t odd_turn = 0;
            if (t < t_end) {
                const TileRuns now = tile_runs(ms.runs, t - c0);
                if constexpr (SCALED) load_scales(now, 0);
                load_k(now);
                load_v(now);
            }
            for (; t < t_end; t += NW) {
                const bool more = t + NW < t_end;
                TileRuns next{};
                if (more) next = tile_runs(ms.runs, t + NW - c0);
                wait_loads<LOADS>();  // (the values', issued behind the keys')

                // ---- scores ----
                float s[NS];
                {
                    Acc<R> x[Ge::NA];
#pragma unroll
                    for (int i = 0; i < Ge::NA; ++i) x[i] = Acc<R>{};
                    if constexpr (ES == 2) {
#pragma unroll
                        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                            for (int i = 0; i < Ge::NA; ++i) {
                                const u32x4 k = lds_at((ktile + key_place<R, RB>(i, lane)) ^ key_step<R>(ks));
#pragma unroll
                                for (int p = NP - 1; p >= 0; --p) x[i] = mfma<CT>(k, q[p][ks], x[i]);
                            }
                    } else {
#pragma unroll
                        for (int k2 = 0; k2 < KS / 2; ++k2)
#pragma unroll
                            for (int i = 0; i < Ge::NA; ++i) {
                                const u32x4 w = lds_at((ktile + key_place<R, RB>(i, lane)) ^ key_step<R>(k2));
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    const u32x2 y = widen<CT>(w[2 * e]), z = widen<CT>(w[2 * e + 1]);
#pragma unroll
                                    for (int p = NP - 1; p >= 0; --p)
                                        x[i] = mfma<CT>(u32x4{y[0], y[1], z[0], z[1]}, q[p][2 * k2 + e], x[i]);
                                }
                            }
                    }
#pragma unroll
                    for (int i = 0; i < NS; ++i) s[i] = x[i / Ge::AE][i % Ge::AE];
                }
                wait_lds();
                if (more) {
                    if constexpr (SCALED) load_scales(next, odd_turn ^ 1);
                    load_k(next);
                }

                // ---- weights ----
                float rf[NS];
                if constexpr (SCALED) {
                    const float *const kfac = raw + 64 * odd_turn;
                    if (lane >= 32) {
                        // (a factor of 0: values of next to nothing; NaN stays)
                        const float y = kfac[lane], x = y == y ? fmaxf(y, 0x1p-126f) : y;
                        lv[lane - 32] = __builtin_amdgcn_logf(x);
                        iv[lane - 32] = __builtin_amdgcn_rcpf(x);
                    }
                    odd_turn ^= 1;
#pragma unroll
                    for (int i = 0; i < NS; i += 4) {
                        const uint32_t tok = token_of_reg<R>(i, g);
                        const f32x4 x = *reinterpret_cast<const f32x4 *>(kfac + tok);
                        const f32x4 y = *reinterpret_cast<const f32x4 *>(lv + tok);
                        const f32x4 z = *reinterpret_cast<const f32x4 *>(iv + tok);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            s[i + j] = fmaf(s[i + j] * factor, x[j], y[j]);
                            rf[i + j] = z[j];
                        }
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < NS; ++i) s[i] *= factor;
                }
                const int32_t j0 = b.lo + 32 * int32_t(t);
                // whether every row sees every token of the tile
                const uint32_t held = tile_held(ms.runs, t - c0);
                const bool full = held == 3 && j0 + 31 <= b.first && (a.window == 0 || int64_t(j0) + a.window > int64_t(b.last));
                uint32_t seen = (1u << NS) - 1;
                if (!full) {
                    seen = 0;
#pragma unroll
                    for (int i = 0; i < NS; ++i) {
                        const uint32_t tok = token_of_reg<R>(i, g);
                        const int32_t j = j0 + int32_t(tok);
                        if (j <= pos && j >= from && (held >> (tok / 16)) & 1) seen |= 1u << i;
                        s[i] = (seen >> i) & 1 ? s[i] : kNegInf;
                    }
                }
                const float tmax = groups_max<R>(max_of(s));
                if (__builtin_expect(__ballot(tmax > m + kLazy) != 0, 0)) {
                    asm volatile("; raise");  // (a branch, not a product by 1 of every sum in every step)
                    const float up = tmax > m + kLazy ? tmax : m;
                    const float al = up == m ? 1.0f : __builtin_amdgcn_exp2f(m - up);
                    m = up;
                    l *= al;
#pragma unroll
                    for (int d = 0; d < DB; ++d) o[d] *= al;
                }
                const float ref = (m == kNegInf ? 0.0f : m) - kLift;
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    s[i] = __builtin_amdgcn_exp2f(s[i] - ref);
                    // (the factor of a token that is not seen may be anything)
                    l += SCALED ? ((seen >> i) & 1 ? s[i] * rf[i] : 0.0f) : s[i];
                }

                // ---- values ----
                if (more)
                    wait_loads<LOADS + (SCALED ? 1 : 0)>();
                else
                    wait_loads<0>();
                bool odd = false;  // values that are not finite where some row must not see them
                if (CT != kI8 && !full) odd = tile_not_finite<CT, Sh::TILE>(mine + Sh::TILE, lane);
                if (!odd) {
                    u32x4 pw[NP];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float x = s[2 * j], y = s[2 * j + 1];
#pragma unroll
                        for (int p = 0; p < NP; ++p) pw[p][j] = piece2<CT>(x, y);
                    }
#pragma unroll
                    for (int d = 0; d < DB; ++d) {
                        u32x4 v;
                        if constexpr (ES == 2) {
                            v = value_frag<RB>((vtile + value_place<R, RB>(lane)) ^ value_block<R>(d), 0);
                        } else {
                            // 8 tokens of one dim: 16 lanes give 8 rows of 16 bytes
                            const uint32_t r = 8 * g + (lane & 15) / 2;
                            const u32x2 w = __builtin_bit_cast(
                                u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32(reinterpret_cast<__attribute__((address_space(3))) s32x2 *>(
                                           vtile + r * RB + ((d ^ value_swizzle<R, RB, 1>(r)) << 4) + 8 * (lane & 1))));
                            const u32x2 x = widen<CT>(w[0]), y = widen<CT>(w[1]);
                            v = u32x4{x[0], x[1], y[0], y[1]};
                        }
#pragma unroll
                        for (int p = NP - 1; p >= 0; --p) o[d] = mfma<CT>(v, pw[p], o[d]);
                    }
                } else {
                    add_values_one_by_one<CT, R, RB, DP>(mine + Sh::TILE, s, seen, lane, o);
                }
                wait_lds();
                if (more) load_v(next);
            }
        }

        // ---- the waves' sums joined ----
        l = groups_sum<R>(l);
        if (g == 0) ms.m[wave][col] = m, ms.l[wave][col] = l;
        __syncthreads();
        float top = kNegInf, all = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) top = fmaxf(top, ms.m[w][col]);
        const float weight = m == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(m - top);
#pragma unroll
        for (int w = 0; w < NW; ++w)
            all += ms.m[w][col] == kNegInf ? ms.l[w][col] : ms.l[w][col] * __builtin_amdgcn_exp2f(ms.m[w][col] - top);
        const bool whole = off == 0 && seg == b.tiles;
        const uint32_t slot = 2 * blockIdx.x + (first_seg ? 0 : 1);
        if (wave == 0 && g == 0) {
            ms.inv[col] = !whole ? 1.0f : all == 0.0f ? 0.0f : 1.0f / all;
            if (!whole) {
                sc.ml[(slot * R + col) * 2] = top;
                sc.ml[(slot * R + col) * 2 + 1] = all;
            }
        }
        // 64 dims at a time: a wave's [16][64] floats in swizzled chunks of 4
#pragma unroll
        for (int d0 = 0; d0 < DB; d0 += 4) {
#pragma unroll
            for (int d = 0; d < 4; ++d) *reinterpret_cast<f32x4 *>(mine + col * 256 + (((4 * d + g) ^ col) << 4)) = o[d0 + d] * weight;
            __syncthreads();
            const uint32_t r = tid / 16, c = tid % 16, e = R * d0 + 4 * c;
            f32x4 x = {0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < NW; ++w)
                x += *reinterpret_cast<const f32x4 *>(lds + Sh::MISC + w * Sh::WAVE + r * 256 + ((c ^ r) << 4));
            if (r0 + r < b.rows) {
                if (!whole)
                    *reinterpret_cast<f32x4 *>(sc.o + (uint64_t(slot) * R + r) * DP + e) = x;
                else if (e < D)
                    store4(a, b.begin, kvh, r0 + r, e, x * ms.inv[r]);
            }
            __syncthreads();
        }
        // this workgroup has the rows' first tiles but not their last: the join is on its list
        if (off == 0 && !whole && tid == 0)
            sc.jobs[blockIdx.x] = SplitJob{seq, r0, kvh, 1 + uint32_t((b.tiles - seg + part - 1) / part), slot};
        left -= seg;
        first_seg = false;
        if (left != 0) next_block<R>(a, rg, b.rows, pl);
    }
}

}  // namespace
}  // namespace tc
