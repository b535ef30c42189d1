// tc_attn_split.hpp -- attention of few rows per key/value head: decode steps and
// drafted tokens. HBM-bound: every cached key and value of a head is read once for
// up to 32 rows.
//
// The line of tiles (32 tokens for 32 rows) is cut into equal parts, one per
// workgroup. The waves of a workgroup take its tiles in turn,
// each through LDS of its own and without barriers: keys of the next tile are on
// their way while the values of this one are multiplied, and the other way round.
// Where a sequence's tiles end or the part does, the waves join their sums. Blocks
// of rows whose tiles lie in several parts leave unnormalised sums, which
// k_attn_join adds up.
#pragma once

#include "tc_attn_kernel.hpp"

namespace tc {
namespace {

// Shape of a launch for one cache type, number of pieces and padded head size.
template <int CT, int NP, int DP>
struct SplitShape {
    static constexpr int ES = scaled_type(CT) ? 1 : 2;
    static constexpr int RB = DP * ES;                       // bytes of a cache row in LDS
    static constexpr int TILE = kTileTokens * RB;            // of a tile of keys or values
    static constexpr int SCALES = scaled_type(CT) ? 768 : 0;  // factors: raw, then log2 and reciprocal
    static constexpr int WAVE = 2 * TILE + SCALES;
    static constexpr int Q = NP * 32 * 2 * DP;
    static constexpr bool QREG = NP * DP <= 256;  // rows of q in registers (64 of them at most)
    // (the first MISC bytes of LDS hold the small things)
    static constexpr int MISC = 8192;
    static constexpr int NW = MISC + (QREG ? 0 : Q) + 4 * WAVE <= 160 * 1024 ? 4 : 3;
    static constexpr int LDS = MISC + (QREG ? (NW * WAVE > Q ? NW * WAVE : Q) : Q + NW * WAVE);
    // workgroups per CU: what LDS and, at this size of the sums, the registers allow
    static constexpr int BY_LDS = 160 * 1024 / LDS;
    static constexpr int OCC = DP == 256 ? (BY_LDS < 2 ? 1 : 2) : BY_LDS < 2 ? 1 : 2;
};

struct SplitMisc {
    float factor[32];
    float m[4][32], l[4][32];
    LineMisc line;
    RunMisc runs;
};
static_assert(sizeof(SplitMisc) <= 8192, "");

template <int CT, int NP, int DP>
__global__ __launch_bounds__((64 * SplitShape<CT, NP, DP>::NW), (SplitShape<CT, NP, DP>::OCC)) void k_attn_split(
    AttnArgs a, RowRange rg, SplitScratch sc) {
    using Sh = SplitShape<CT, NP, DP>;
    constexpr int ES = Sh::ES, RB = Sh::RB, NW = Sh::NW, KS = DP / 16, DB = DP / 32;
    constexpr bool SCALED = scaled_type(CT);
    extern __shared__ __align__(1024) unsigned char lds[];
    SplitMisc &ms = *reinterpret_cast<SplitMisc *>(lds);
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t col = lane & 31, half = lane >> 5;
    unsigned char *const qlds = lds + Sh::MISC;
    unsigned char *const mine = qlds + (Sh::QREG ? 0 : Sh::Q) + wave * Sh::WAVE;
    unsigned char *const ktile = mine, *const vtile = mine + Sh::TILE;
    float *const raw = reinterpret_cast<float *>(mine + 2 * Sh::TILE);  // [64] factors of keys, of values
    float *const lv = raw + 64, *const iv = raw + 96;                   // [32] log2 and reciprocal of the values'
    const uint32_t kvh_n = a.kv.kv_heads, D = a.kv.dim, rowbytes = D * ES, nch = rowbytes / 16;

    // ---- this workgroup's part of the line of tiles ----
    uint64_t part, left;
    Place pl = line_part<32, kTileTokens, 64 * NW>(a, rg, blockIdx.x, gridDim.x, NW, ms.line, tid, &part, &left);
    if (tid == 0) sc.jobs[blockIdx.x].count = 0;

    bool first_seg = true;
    while (left != 0) {
        const uint32_t seq = pl.seq, r0 = pl.r0, kvh = pl.kvh, off = pl.off;
        const RowBlock b = row_block<32, kTileTokens>(a, seq, r0);
        const uint32_t seg = uint32_t(min(uint64_t(b.tiles - off), left));

        // ---- rows of q ----
        __syncthreads();
        if (tid < 128) stage_q<CT, NP, DP, 128>(a, b.begin, kvh, r0, b.rows, qlds, ms.factor, tid);
        __syncthreads();
        const float factor = ms.factor[col];
        auto q_chunk = [&](int p, int ks) __attribute__((always_inline)) {
            constexpr uint32_t QB = 2 * DP;
            const uint32_t c = step_dim<ES>(ks, half) / 8;
            return *reinterpret_cast<const u32x4 *>(qlds + (p * 32 + col) * QB + ((c ^ key_swizzle<QB>(col)) << 4));
        };
        u32x4 qreg[Sh::QREG ? NP : 1][Sh::QREG ? KS : 1];
        if constexpr (Sh::QREG) {
#pragma unroll
            for (int p = 0; p < NP; ++p)
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) qreg[p][ks] = q_chunk(p, ks);
            __syncthreads();  // (the tiles take the place of the staged rows)
        }
        if (DP != D)  // dims past the row's: zeros, which no load touches
            for (uint32_t i = lane; i < 2 * Sh::TILE / 16; i += 64) *reinterpret_cast<u32x4 *>(mine + 16 * i) = u32x4{0, 0, 0, 0};
        const uint32_t row = r0 + col;
        const int32_t pos = row < b.rows ? b.pos0 + int32_t(row / a.group) : -1;  // the lane's row sees tokens up to here
        const int32_t from = a.window != 0 && int64_t(pos) + 1 > int64_t(a.window) ? int32_t(pos + 1 - a.window) : 0;

        // ---- tiles ----
        const uint32_t run_bytes = 16 * rowbytes;
        constexpr int LPR = RB / 16, RPI = 64 / LPR;  // lanes per row, rows per load
        constexpr int LOADS = 2 * (16 / RPI);         // loads of a tile of keys or values
        auto load = [&](unsigned char *dst, const uint8_t *src, const TileRuns &w, auto swizzle) __attribute__((always_inline)) {
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const uint8_t *from = src + uint64_t(w.run[g]) * run_bytes;
#pragma unroll
                for (int j = 0; j < 16 / RPI; ++j) {
                    const uint32_t r = j * RPI + lane / LPR, c = (lane % LPR) ^ swizzle(16 * g + r);
                    if (DP == D || c < nch) dma16(lds_addr(dst + (16 * g + j * RPI) * RB), from, r * rowbytes + 16 * c);
                }
            }
        };
        auto load_k = [&](const TileRuns &w) __attribute__((always_inline)) {
            load(ktile, a.kv.k, w, key_swizzle<RB>);
        };
        auto load_v = [&](const TileRuns &w) __attribute__((always_inline)) {
            load(vtile, a.kv.v, w, value_swizzle<RB, ES>);
        };
        // lanes 0-31 the keys' factors of the 32 tokens, the others the values'
        auto load_scales = [&](const TileRuns &w) __attribute__((always_inline)) {
            return (half ? a.kv.vs : a.kv.ks)[16 * uint64_t(col >> 4 ? w.run[1] : w.run[0]) + (col & 15)];
        };

        v16f o[DB];
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
        float m = kNegInf, l = 0.0f;

        for (uint32_t c0 = off; c0 < off + seg; c0 += kStretch) {
        const uint32_t t_end = min(off + seg, c0 + kStretch);
        __syncthreads();
        if (tid == 0) ms.runs.missing = 0;
        __syncthreads();
        find_runs<64 * NW>(a, seq, kvh, b.lo + 32 * int32_t(c0), b.hi, t_end - c0, ms.runs, tid);
        __syncthreads();
        uint32_t t = c0 + wave;
        TileRuns now{};
        float next_scale = 0.0f;
        if (t < t_end) {
            now = tile_runs(ms.runs, t - c0);
            wait_lds();
            load_k(now);
            load_v(now);
            if constexpr (SCALED) next_scale = load_scales(now);
        }
        for (; t < t_end; t += NW) {
            const bool more = t + NW < t_end;
            TileRuns next = now;
            if (more) next = tile_runs(ms.runs, t + NW - c0);
            if constexpr (SCALED) {
                raw[lane] = next_scale;
                const float vsc = fmaxf(next_scale, 0x1p-126f);  // (a factor of 0: values of next to nothing)
                const float x = vsc == vsc ? vsc : next_scale;
                if (half) {
                    lv[col] = __builtin_amdgcn_logf(x);
                    iv[col] = __builtin_amdgcn_rcpf(x);
                }
                if (next_scale != next_scale && half) lv[col] = next_scale;
            }
            // keys: the last loads but the values'
            wait_loads<LOADS>();
            v16f s;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = 0.0f;
            {
                const uint32_t r = token_of_row(col);
                const unsigned char *kr = ktile + r * RB;
                if constexpr (ES == 2) {
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) {
                        const u32x4 k = *reinterpret_cast<const u32x4 *>(kr + (((2 * ks + half) ^ key_swizzle<RB>(r)) << 4));
#pragma unroll
                        for (int p = NP - 1; p >= 0; --p) s = mfma<CT>(k, Sh::QREG ? qreg[p][ks] : q_chunk(p, ks), s);
                    }
                } else {
#pragma unroll
                    for (int k2 = 0; k2 < KS / 2; ++k2) {
                        const u32x4 w = *reinterpret_cast<const u32x4 *>(kr + (((2 * k2 + half) ^ key_swizzle<RB>(r)) << 4));
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const u32x2 x = widen<CT>(w[2 * e]), y = widen<CT>(w[2 * e + 1]);
#pragma unroll
                            for (int p = NP - 1; p >= 0; --p)
                                s = mfma<CT>(u32x4{x[0], x[1], y[0], y[1]},
                                             Sh::QREG ? qreg[p][2 * k2 + e] : q_chunk(p, 2 * k2 + e), s);
                        }
                    }
                }
            }
            wait_lds();
            if (more) load_k(next);

            // ---- weights ----
            float kf[16], lf[16], rf[16];
            if constexpr (SCALED) {
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const uint32_t tok = token_of_reg(i, half);
                    const f32x4 x = *reinterpret_cast<const f32x4 *>(raw + tok);
                    const f32x4 y = *reinterpret_cast<const f32x4 *>(lv + tok);
                    const f32x4 z = *reinterpret_cast<const f32x4 *>(iv + tok);
#pragma unroll
                    for (int j = 0; j < 4; ++j) kf[i + j] = x[j], lf[i + j] = y[j], rf[i + j] = z[j];
                }
            }
            const int32_t j0 = b.lo + 32 * int32_t(t);
            // whether every row of the block sees every token of the tile
            const bool full = now.held == 3 && j0 + 31 <= b.first && (a.window == 0 || int64_t(j0) + a.window > int64_t(b.last));
            uint32_t seen = 0xFFFF;
            if (!full) {
                seen = 0;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int32_t j = j0 + int32_t(token_of_reg(i, half));
                    if (j <= pos && j >= from && (now.held >> (i / 8)) & 1) seen |= 1u << i;
                }
            }
            float tmax;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float x = s[i] * factor;
                if constexpr (SCALED) x = fmaf(x, kf[i], lf[i]);
                if (!full) x = (seen >> i) & 1 ? x : kNegInf;
                s[i] = x;
            }
            tmax = halves_max(max16(s));
            if (__ballot(tmax > m + kLazy) != 0) {
                const float up = tmax > m + kLazy ? tmax : m;
                const float al = up == m ? 1.0f : __builtin_amdgcn_exp2f(m - up);
                m = up;
                l *= al;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[d][i] *= al;
            }
            const float ref = (m == kNegInf ? 0.0f : m) - kLift;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float p = __builtin_amdgcn_exp2f(s[i] - ref);
                s[i] = p;
                if constexpr (SCALED)
                    l += (seen >> i) & 1 ? p * rf[i] : 0.0f;
                else
                    l += p;
            }

            // ---- values ----
            if (more)
                wait_loads<LOADS>();
            else
                wait_loads<0>();
            bool odd = false;  // values that are not finite where some row must not see them
            if (CT != kI8 && !full) odd = tile_not_finite<CT, Sh::TILE>(vtile, lane);
            if (!odd) {
                // P^T of 16 tokens: the registers as they are
                u32x4 pw[2][NP];
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float x = s[8 * k + 2 * j], y = s[8 * k + 2 * j + 1];
#pragma unroll
                        for (int p = 0; p < NP; ++p) pw[k][p][j] = piece2<CT>(x, y);
                    }
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        u32x4 v;
                        if constexpr (ES == 2) {
                            v = value_frag<RB>(lds_addr(vtile) + value_place<RB>(d, lane), k);
                        } else {
                            const uint32_t l16 = lane & 15, g16 = (lane >> 4) & 1;
                            const uint32_t r = 16 * k + 8 * half + l16 / 2, e = 32 * d + 16 * g16 + 8 * (l16 % 2);
                            const unsigned char *p = vtile + r * RB + (((e / 16) ^ value_swizzle<RB, ES>(r)) << 4) + (e & 8);
                            const u32x2 w = __builtin_bit_cast(
                                u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) s32x2 *)(p)));
                            const u32x2 x = widen<CT>(w[0]), y = widen<CT>(w[1]);
                            v = u32x4{x[0], x[1], y[0], y[1]};
                        }
#pragma unroll
                        for (int p = NP - 1; p >= 0; --p) o[d] = mfma<CT>(v, pw[k][p], o[d]);
                    }
            } else {
                add_values_one_by_one<CT, RB, DB>(vtile, s, seen, lane, o);
            }
            wait_lds();
            if (more) {
                load_v(next);
                if constexpr (SCALED) next_scale = load_scales(next);
            }
            now = next;
        }
        }

        // ---- the waves' sums joined ----
        l = halves_sum(l);
        if (half == 0) ms.m[wave][col] = m, ms.l[wave][col] = l;
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
        if (!whole && wave == 0 && half == 0) {
            sc.ml[(slot * 32 + col) * 2] = top;
            sc.ml[(slot * 32 + col) * 2 + 1] = all;
        }
        const float inv = all == 0.0f ? 0.0f : 1.0f / all;
#pragma unroll
        for (int d = 0; d < DB; ++d) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                f32x4 x;
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = o[d][4 * k + j] * weight;
                *reinterpret_cast<f32x4 *>(mine + col * 128 + (((2 * k + half) ^ (col & 7)) << 4)) = x;
            }
            if (half == 0 && wave == 0) ms.factor[col] = whole ? inv : 1.0f;
            __syncthreads();
            for (uint32_t i = tid; i < 256; i += 64 * NW) {
                const uint32_t r = i / 8, c = i % 8, e = 32 * d + 4 * c;
                f32x4 x = {0, 0, 0, 0};
#pragma unroll
                for (int w = 0; w < NW; ++w)
                    x += *reinterpret_cast<const f32x4 *>(mine + (int(w) - int(wave)) * Sh::WAVE + r * 128 + ((c ^ (r & 7)) << 4));
                const uint32_t row = r0 + r;
                if (row < b.rows) {
                    if (!whole) {
                        *reinterpret_cast<f32x4 *>(sc.o + (uint64_t(slot) * 32 + r) * DP + e) = x;
                    } else if (e < D) {
                        const float f = ms.factor[r];
                        store4(a, b.begin, kvh, row, e, x * f);
                    }
                }
            }
            __syncthreads();
        }
        // this workgroup has the block's first tiles but not its last: the join is on its list
        if (off == 0 && !whole && tid == 0)
            sc.jobs[blockIdx.x] = SplitJob{seq, r0, kvh, 1 + uint32_t((b.tiles - seg + part - 1) / part), slot};

        left -= seg;
        first_seg = false;
        if (left != 0) next_block<32>(a, rg, b.rows, pl);
    }
}

}  // namespace
}  // namespace tc
