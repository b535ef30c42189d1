// tc_attn_few.hpp -- attention of up to kFewRows rows per key/value head: decode steps
// and drafted tokens. HBM-bound: every cached key and value of a head is read once for
// 16 rows.
//
// The waves of a workgroup take the tiles of its part (32 tokens for 16 rows) in turn,
// each through LDS of its own and without barriers: while one tile is multiplied, the
// keys and values of the next ones are on their way. Where a block's tiles end or the
// part does, the waves join their sums. Blocks whose tiles lie in several parts leave
// unnormalised sums, which k_attn_join adds up.
//
// Up to 16 KB of tiles per wave are on their way, 128 KB per CU, in LDS directly, so
// that neither registers nor a barrier bound them. 8 waves, not 4, together with one launch
// for a batch of any mix: 61 -> 35 us for 16 sequences of drafted tokens. Rows of 16, not
// 32: 20 -> 16 us for one token at 1000.
// Measured: 64 decoding sequences (bf16, 8 heads of 128, 1.04 GB) 166 us, 6.3 TB/s; one
// token at 131071 (int8, 138 MB) 38 us, 3.6 TB/s, of which 6 are the join and about as
// many the start and the blocks' sums; one token at 1001 (2 MB) 13.8 us: launches, 3.5 us
// until a workgroup knows its part, and what the first instructions and rows take to arrive.
#pragma once

#include "tc_attn_kernel.hpp"

namespace tc {
namespace {

template <int CT, int NP, int DP>
struct FewShape {
    static constexpr int R = 16;
    static constexpr int ES = scaled_type(CT) ? 1 : 2;
    static constexpr int RB = DP * ES;             // bytes of a cache row in LDS
    static constexpr int TILE = kTileTokens * RB;  // of a tile of keys or values
    // tiles in flight per wave, and waves at work: 16 KB each, or 4 of 32
    static constexpr int NB = 2 * TILE <= 16384 ? 16384 / (2 * TILE) : 1;
    static constexpr int NW = 2 * TILE <= 16384 ? kWaves : 4;
    static constexpr int SCALES = scaled_type(CT) ? 256 * (NB + 2) : 0;  // factors of NB + 1 tiles; log2 and reciprocal
    static constexpr int WAVE = 2 * TILE * NB + SCALES;
    static constexpr int START = 12;  // places of a block without a tile
    static constexpr int LDS = kMisc + NW * WAVE;
    static_assert(LDS <= kLds, "");
};

template <int CT, int NP, int DP, int SLOT>
__device__ __forceinline__ void attn_few(const AttnArgs &a, RowRange rg, Seqs seqs, const SplitScratch &sc, Part work, unsigned char *lds, Misc &ms) {
    using Sh = FewShape<CT, NP, DP>;
    constexpr int R = Sh::R, ES = Sh::ES, RB = Sh::RB, NW = Sh::NW, NB = Sh::NB, TILE = Sh::TILE;
    using Ge = Geo<R, DP>;
    constexpr int KS = Ge::KS, DB = Ge::DB, NS = Ge::NS;
    constexpr bool SCALED = scaled_type(CT);
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t col = lane % R, g = lane / R;
    // LDS of the wave: NB tiles of keys, NB of values, factors (waves without work: the last one's)
    unsigned char *const mine = lds + kMisc + min(wave, NW - 1u) * Sh::WAVE;
    const uint32_t kring = lds_addr(lds) + kMisc + min(wave, NW - 1u) * Sh::WAVE, vring = kring + NB * TILE;
    float *const raw = reinterpret_cast<float *>(mine + 2 * NB * TILE);       // [NB + 1][64] a tile's factors: keys', values'
    float *const lv = raw + 64 * (NB + 1), *const iv = lv + 32;               // [32] log2 and reciprocal of the values'
    const uint32_t D = a.kv.dim, rowbytes = D * ES, run_bytes = 16 * rowbytes, nch = rowbytes / 16;

    // (as for many rows: formed anew, not kept, where registers are short)
    constexpr bool SHORT = NP * DP >= 512;
    auto place_lane = [&]() __attribute__((always_inline)) { return SHORT ? lane_now() : lane; };

    Place pl = work.at;
    uint64_t left = work.left;
    bool first_seg = true;
    while (left != 0) {
        const uint32_t seq = pl.seq, r0 = pl.r0, kvh = pl.kvh;
        const RowBlock b = row_block<R, kTileTokens>(a, seqs.uniform(a, seq), r0);
        const Segment sg = segment<Sh::START>(b.tiles, pl.off, left);
        const uint32_t off = sg.off, seg = sg.tiles;
        if (seg == 0) break;  // (the part ends among the block's first places)

        const uint32_t row = r0 + col;
        u32x4 raw_q[f32_rows<CT, NP>() ? 2 : 1][KS], q[NP][KS];
        fetch_q<CT, NP, R, DP, ES>(a, b.begin, kvh, row, b.rows, g, raw_q);
        find_runs<kThreads>(a, seq, kvh, b.lo + 32 * int32_t(off), b.last, min(seg, 512u), ms.runs, tid);
        __syncthreads();
        const float factor = make_q<CT, NP, R, DP>(a, raw_q, q);
        const int32_t pos = row < b.rows ? b.pos0 + int32_t(div_fast(row, a.group_div)) : -1;  // the lane's row sees tokens up to here
        const int32_t from = max(0, max(pos, -1) + 1 - a.span);

        constexpr int LPR = RB / 16, RPI = 64 / LPR;  // lanes per row, rows per load
        constexpr int LOADS = 2 * (16 / RPI);         // loads of a tile of keys or values
        // (lines that no other block reads are the first that the caches give up: 64
        // decoding sequences 198 -> 175 us, while 4 blocks read 5% slower so)
        const bool once = b.rows <= R;
        auto load = [&](uint32_t dst, const uint8_t *src, const TileRuns &w, auto swizzle) __attribute__((always_inline)) {
            const uint32_t ln = place_lane();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint8_t *at = src + uint64_t(w.of(h != 0)) * run_bytes;
#pragma unroll
                for (int j = 0; j < 16 / RPI; ++j) {
                    const uint32_t r = j * RPI + ln / LPR, c = (ln % LPR) ^ swizzle(16 * h + r);
                    // (dims past the row's: others of it, which meet zeros of q, or go nowhere)
                    const uint32_t lane_off = r * rowbytes + (c < nch ? 16 * c : 0);
                    if (once)
                        dma16<true>(dst + (16 * h + j * RPI) * RB, at, lane_off);
                    else
                        dma16<false>(dst + (16 * h + j * RPI) * RB, at, lane_off);
                }
            }
        };
        // tile number i of the wave
        auto load_k = [&](const TileRuns &w, uint32_t i) __attribute__((always_inline)) {
            load(kring + i % NB * TILE, a.kv.k, w, key_swizzle<R, RB>);
        };
        auto load_v = [&](const TileRuns &w, uint32_t i) __attribute__((always_inline)) {
            load(vring + i % NB * TILE, a.kv.v, w, value_swizzle<R, RB, ES>);
        };
        // lanes 0-31 the keys' factors of the 32 tokens, the others the values'
        auto load_scales = [&](const TileRuns &w, uint32_t i) __attribute__((always_inline)) {
            const float *p = lane >= 32 ? a.kv.vs : a.kv.ks;
            dma4(kring + 2 * NB * TILE + i % (NB + 1) * 256, p + 16 * uint64_t(w.of(lane & 16)) + (lane & 15));
        };

        Acc<R> o[DB];
#pragma unroll
        for (int d = 0; d < DB; ++d) o[d] = Acc<R>{};
        float m = kNegInf, l = 0.0f;

        for (uint32_t c0 = off; c0 < off + seg; c0 += 512) {
            const uint32_t t_end = min(off + seg, c0 + 512);
            if (c0 != off) {
                __syncthreads();
                find_runs<kThreads>(a, seq, kvh, b.lo + 32 * int32_t(c0), b.last, t_end - c0, ms.runs, tid);
                __syncthreads();
            }
            const uint32_t mine_n = wave < uint32_t(NW) && t_end - c0 > wave ? (t_end - c0 - wave + NW - 1) / NW : 0;  // the wave's tiles
            wait_lds();
#pragma unroll
            for (uint32_t i = 0; i < NB; ++i)
                if (i < mine_n) {
                    const TileRuns w = tile_runs(ms.runs, wave + NW * i);
                    if constexpr (SCALED) load_scales(w, i);
                    load_k(w, i);
                    load_v(w, i);
                }
            for (uint32_t n = 0; n < mine_n; ++n) {
                const uint32_t t = c0 + wave + NW * n;
                const uint32_t ktile = kring + n % NB * TILE, vtile = vring + n % NB * TILE;
                const bool more = n + NB < mine_n;
                TileRuns next{};
                if (more) next = tile_runs(ms.runs, t + NW * NB - c0);
                // (all loads behind the keys', where NB - 1 further tiles are under way)
                if (n + NB <= mine_n)
                    wait_loads<(2 * NB - 1) * LOADS + (SCALED ? NB - 1 : 0)>();
                else
                    wait_loads<0>();

                // ---- scores ----
                float s[NS];
                {
                    const uint32_t ln = place_lane();
                    Acc<R> x[Ge::NA];
#pragma unroll
                    for (int i = 0; i < Ge::NA; ++i) x[i] = Acc<R>{};
                    if constexpr (ES == 2) {
#pragma unroll
                        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                            for (int i = 0; i < Ge::NA; ++i) {
                                const u32x4 k = lds_at((ktile + key_place<R, RB>(i, ln)) ^ key_step<R>(ks));
#pragma unroll
                                for (int p = NP - 1; p >= 0; --p) x[i] = mfma<CT>(k, q[p][ks], x[i]);
                            }
                    } else {
#pragma unroll
                        for (int k2 = 0; k2 < KS / 2; ++k2)
#pragma unroll
                            for (int i = 0; i < Ge::NA; ++i) {
                                const u32x4 w = lds_at((ktile + key_place<R, RB>(i, ln)) ^ key_step<R>(k2));
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
                    if constexpr (SCALED) load_scales(next, n + NB);
                    load_k(next, n + NB);
                }

                // ---- weights ----
                float rf[NS], vfac = 0.0f;
                if constexpr (SCALED) {
                    const float *const kfac = raw + n % (NB + 1) * 64;
                    if (lane >= 32) {
                        vfac = kfac[lane];
                        const float x = value_factor(vfac);
                        lv[lane - 32] = __builtin_amdgcn_logf(x);
                        iv[lane - 32] = __builtin_amdgcn_rcpf(x);
                    }
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
                const bool full = held == 3 && j0 + 31 <= b.first && int64_t(j0) + a.span > int64_t(b.last);
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
                float tmax = groups_max<R>(max_of(s));
                if (__builtin_expect(__ballot(tmax > m + kLazy) != 0, 0)) {
                    asm volatile("; raise");  // (a branch, not a product by 1 of every sum in every step)
                    uint32_t zeros = 0;
                    if constexpr (SCALED) {
                        const uint32_t ones = uint32_t(__ballot(vfac == 1.0f) >> 32);
                        if (__builtin_expect(ones != 0, 0)) {
                            wait_loads<0>();  // (the tile's values are still on their way)
                            zeros = rows_of_zeros<CT, RB>(ones, mine + (NB + n % NB) * TILE, lane_now());
                        }
                        if (__builtin_expect(zeros != 0, 0)) {
                            lower_zeros<R>(s, zeros, g);
                            tmax = groups_max<R>(max_of(s));
                        }
                    }
                    const float up = tmax > m + kLazy ? tmax : m;
                    const float al = up == m ? 1.0f : __builtin_amdgcn_exp2f(m - up);
                    m = up;
                    l *= al;
#pragma unroll
                    for (int d = 0; d < DB; ++d) o[d] *= al;
                    if constexpr (SCALED)
                        if (__builtin_expect(zeros != 0, 0)) l += take_zeros<R>(s, zeros, g, (m == kNegInf ? 0.0f : m) - kLift);
                }
                const float ref = (m == kNegInf ? 0.0f : m) - kLift;
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    s[i] = __builtin_amdgcn_exp2f(s[i] - ref);
                    // (the factor of a token that is not seen may be anything)
                    if constexpr (SCALED)
                        l += (seen >> i) & 1 ? s[i] * rf[i] : 0.0f;
                    else if constexpr (!rounded_sum<CT, NP>())
                        l += s[i];
                }

                // ---- values ----
                if (more)
                    wait_loads<(2 * NB - 1) * LOADS + (SCALED ? NB : 0)>();
                else
                    wait_loads<0>();
                bool odd = false;  // values that are not finite where some row must not see them
                if (CT != kI8 && !full) odd = tile_not_finite<CT, TILE>(mine + (NB + n % NB) * TILE, lane);
                if (!odd) {
                    u32x4 pw[NP];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float x = s[2 * j], y = s[2 * j + 1];
#pragma unroll
                        for (int p = 0; p < NP; ++p) pw[p][j] = piece2<CT>(x, y);
                        if constexpr (rounded_sum<CT, NP>()) l = add_pair<CT>(pw[0][j], l);
                    }
                    const uint32_t ln = place_lane();
#pragma unroll
                    for (int d = 0; d < DB; ++d) {
                        u32x4 v;
                        if constexpr (ES == 2) {
                            v = value_frag<RB>((vtile + value_place<R, RB>(ln)) ^ value_block<R>(d), 0);
                        } else {
                            // 8 tokens of one dim: 16 lanes give 8 rows of 16 bytes
                            const uint32_t r = 8 * (ln / R) + (ln & 15) / 2;
                            const u32x2 w = __builtin_bit_cast(
                                u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32(reinterpret_cast<__attribute__((address_space(3))) s32x2 *>(
                                           vtile + r * RB + ((d ^ value_swizzle<R, RB, 1>(r)) << 4) + 8 * (ln & 1))));
                            const u32x2 x = widen<CT>(w[0]), y = widen<CT>(w[1]);
                            v = u32x4{x[0], x[1], y[0], y[1]};
                        }
#pragma unroll
                        for (int p = NP - 1; p >= 0; --p) o[d] = mfma<CT>(v, pw[p], o[d]);
                    }
                } else {
                    if constexpr (rounded_sum<CT, NP>())
#pragma unroll
                        for (int i = 0; i < NS; ++i) l += s[i];
                    add_values_one_by_one<CT, R, RB, DP>(mine + (NB + n % NB) * TILE, s, seen, lane, o);
                }
                wait_lds();
                if (more) load_v(next, n + NB);
            }
        }

        // ---- the waves' sums joined ----
        l = groups_sum<R>(l);
        if (g == 0 && wave < uint32_t(NW)) ms.few.m[wave][col] = m, ms.few.l[wave][col] = l;
        __syncthreads();
        float top = kNegInf, all = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) top = fmaxf(top, ms.few.m[w][col]);
        const float weight = m == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(m - top);
#pragma unroll
        for (int w = 0; w < NW; ++w)
            all += ms.few.m[w][col] == kNegInf ? ms.few.l[w][col] : ms.few.l[w][col] * __builtin_amdgcn_exp2f(ms.few.m[w][col] - top);
        const bool whole = off == 0 && seg == b.tiles;
        const uint32_t slot = 2 * work.id + (first_seg ? 0 : 1);
        if (wave == 0 && g == 0) {
            ms.few.inv[col] = !whole ? 1.0f : all == 0.0f ? 0.0f : 1.0f / all;
            if (!whole) {
                sc.ml[(slot * SLOT + col) * 2] = top;
                sc.ml[(slot * SLOT + col) * 2 + 1] = all;
            }
        }
        // up to 128 dims at a time: a wave's [16][128] floats in swizzled chunks of 4
        constexpr int DS = DB < 8 ? DB : 8;
#pragma unroll
        for (int d0 = 0; d0 < DB; d0 += DS) {
            if (wave < uint32_t(NW))
#pragma unroll
                for (int d = 0; d < DS; ++d)
                    *reinterpret_cast<f32x4 *>(mine + col * 64 * DS + (((4 * d + g) ^ col) << 4)) = o[d0 + d] * weight;
            __syncthreads();
            const uint32_t r = tid / (4 * DS), c = tid % (4 * DS), e = R * d0 + 4 * c;
            if (r0 + r < b.rows && r < R) {
                f32x4 x = {0, 0, 0, 0};
#pragma unroll
                for (int w = 0; w < NW; ++w)
                    x += *reinterpret_cast<const f32x4 *>(lds + kMisc + w * Sh::WAVE + r * 64 * DS + ((c ^ r) << 4));
                if (!whole)
                    *reinterpret_cast<f32x4 *>(sc.o + (uint64_t(slot) * SLOT + r) * DP + e) = x;
                else if (e < D)
                    store4(a, b.begin, kvh, r0 + r, e, x * ms.few.inv[r]);
            }
            __syncthreads();
        }
        // this workgroup has the rows' first tiles but not their last: the join is on its list
        if (off == 0 && !whole && tid == 0)
            sc.jobs[work.id] = SplitJob{b.begin, r0, kvh, min(uint32_t(R), b.rows - r0), 1 + uint32_t((b.tiles - seg + work.part - 1) / work.part), slot};
        left -= sg.places;
        first_seg = false;
        if (left != 0 && !next_block<R>(a, rg, seqs, b.rows, pl)) break;
    }
}

}  // namespace
}  // namespace tc
