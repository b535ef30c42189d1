// tc_attn_many.hpp -- attention of many rows per key/value head: prompts. Bound by
// the matrix cores and the exponentials between their products.
//
// A workgroup takes 32 (or 16) rows per wave of one key/value head, which go over its tiles
// of 32 tokens together: tiles come into LDS two steps ahead (8-bit ones through
// registers, widened to fp16 once for all waves), rows of q stay in registers. A
// step's score products belong to the tile behind the one whose weights are being
// formed, so that a wave's matrix and vector work do not wait for each other. The
// line of tiles is cut into one part per CU; blocks that a cut goes through leave
// their sums for k_attn_join.
//
// Measured: 2048 rows of 28 heads of 128 at 8193 tokens (bf16, 210 GFLOP) 230 to 245 us,
// 860 to 915 TFLOP/s, where a large library product reaches 1190: matrix cores busy 41%
// of the time, vector instructions 39%, no LDS conflicts; the two of a SIMD hardly overlap
// although their order is pinned side by side. As fast: two workgroups of 4 waves per
// CU; a barrier between the two products. Slower: a barrier at every second tile (247
// against 241). Seven sequences of fp32 rows (two pieces) over int8 heads of 256, 127 us.
#pragma once

#include <type_traits>

#include "tc_attn_kernel.hpp"

namespace tc {
namespace {

template <int CT, int NP, int DP>
struct ManyShape {
    static constexpr int LT = CT == kBF16 ? kBF16 : kF16;  // element type in LDS
    static constexpr int RB = 2 * DP;
    static constexpr int TILE = kTileTokens * RB;
    // 32 rows per wave where the sums and q leave room in the registers, else 16
    static constexpr int R = NP == 1 && DP <= 128 ? 32 : 16;
    static constexpr int ROWS = R * kWaves;
    static constexpr int NBUF = 4;
    static constexpr int START = 20;  // places of a block without a tile
    static constexpr int LDS = kMisc + 2 * NBUF * TILE;
};

__device__ __forceinline__ void tile_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <int CT, int NP, int DP, int SLOT>
__device__ __forceinline__ void attn_many(const AttnArgs &a, RowRange rg, Seqs seqs, const SplitScratch &sc, Part work, unsigned char *lds, Misc &ms) {
    using Sh = ManyShape<CT, NP, DP>;
    constexpr int R = Sh::R, LT = Sh::LT, RB = Sh::RB, NW = kWaves, TILE = Sh::TILE, NBUF = Sh::NBUF, STRETCH = 512;
    using Ge = Geo<R, DP>;
    constexpr int KS = Ge::KS, DB = Ge::DB, NS = Ge::NS, NA = Ge::NA, AE = Ge::AE;
    constexpr uint32_t ALL = (1u << NS) - 1;
    constexpr bool SCALED = scaled_type(CT);
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t col = lane % R, g = lane / R;
    const uint32_t kbuf = lds_addr(lds) + kMisc, vbuf = kbuf + NBUF * TILE;
    const uint32_t D = a.kv.dim, rowbytes = D * (SCALED ? 1 : 2);

    // Where rows of q in several pieces and wide sums fill the registers, what a tile's loads
    // need of the lane is formed for each: kept, it was spilled, and a reload waits for the
    // tiles on their way (7 sequences, fp32 rows, int8 heads of 256: 157 -> 125 us; narrower
    // ones lose up to 5% so). Fewer operands are fetched ahead there too.
    constexpr bool SHORT = NP * DP >= 512;
    auto place_lane = [&]() __attribute__((always_inline)) { return SHORT ? lane_now() : lane; };

    Place pl = work.at;
    uint64_t left = work.left;
    bool first_seg = true;
    while (left != 0) {
        const uint32_t seq = pl.seq, r0 = pl.r0, kvh = pl.kvh;
        const RowBlock b = row_block<Sh::ROWS, kTileTokens>(a, seqs.uniform(a, seq), r0);
        const Segment sg = segment<Sh::START>(b.tiles, pl.off, left);
        const uint32_t off = sg.off, seg = sg.tiles;
        if (seg == 0) break;  // (the part ends among the block's first places)

        // ---- the wave's rows of q ----
        const uint32_t wr0 = r0 + R * wave, row = wr0 + col;
        const bool active = wr0 < b.rows;  // the wave has rows
        const int32_t pos = row < b.rows ? b.pos0 + int32_t(div_fast(row, a.group_div)) : -1;  // the lane's row sees tokens up to here
        const int32_t from = max(0, max(pos, -1) + 1 - a.span);
        const int32_t wfirst = b.pos0 + int32_t(div_fast(wr0, a.group_div));
        const int32_t wlast = b.pos0 + int32_t(div_fast(min(wr0 + R, b.rows) - 1, a.group_div));
        u32x4 raw_q[f32_rows<CT, NP>() ? 2 : 1][KS], q[NP][KS];
        fetch_q<CT, NP, R, DP, 2>(a, b.begin, kvh, row, b.rows, g, raw_q);
        find_runs<kThreads>(a, seq, kvh, b.lo + 32 * int32_t(off), b.last, min(seg, uint32_t(STRETCH)), ms.runs, tid);
        __syncthreads();
        const float factor = make_q<CT, NP, R, DP>(a, raw_q, q);
        Acc<R> o[DB];
#pragma unroll
        for (int d = 0; d < DB; ++d) o[d] = Acc<R>{};
        float s[NS];
#pragma unroll
        for (int i = 0; i < NS; ++i) s[i] = 0.0f;
        float m = kNegInf, l = 0.0f, tmax = kNegInf;
        uint32_t seen = ALL;

        uint32_t kplace[NA], vplace = vbuf + value_place<R, RB>(lane);
#pragma unroll
        for (int i = 0; i < NA; ++i) kplace[i] = kbuf + key_place<R, RB>(i, lane);
        // scores of the tile in a buffer
        auto products = [&](uint32_t buf, float (&x)[NS]) __attribute__((always_inline)) {
            Acc<R> y[NA];
            uint32_t place[NA];
#pragma unroll
            for (int i = 0; i < NA; ++i) y[i] = Acc<R>{}, place[i] = here(kplace[i]);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int i = 0; i < NA; ++i) {
                    const u32x4 k = lds_at((place[i] ^ key_step<R>(ks)) + buf * TILE);
#pragma unroll
                    for (int p = NP - 1; p >= 0; --p) y[i] = mfma<LT>(k, q[p][ks], y[i]);
                }
#pragma unroll
            for (int i = 0; i < NS; ++i) x[i] = y[i / AE][i % AE];
        };
        // o += weights * values of the tile in a buffer (and l += rounded weights)
        auto add_values = [&](uint32_t buf) __attribute__((always_inline)) {
            u32x4 pw[Ge::KT][NP];
#pragma unroll
            for (int k = 0; k < Ge::KT; ++k)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float x = s[8 * k + 2 * j], y = s[8 * k + 2 * j + 1];
#pragma unroll
                    for (int p = 0; p < NP; ++p) pw[k][p][j] = piece2<LT>(x, y);
                    if constexpr (rounded_sum<CT, NP>()) l = add_pair<LT>(pw[k][0][j], l);
                }
            const uint32_t place = here(vplace);
#pragma unroll
            for (int k = 0; k < Ge::KT; ++k)
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    const u32x4 v = value_frag<RB>((place ^ value_block<R>(d)) + buf * TILE, k);
#pragma unroll
                    for (int p = NP - 1; p >= 0; --p) o[d] = mfma<LT>(v, pw[k][p], o[d]);
                }
        };

        for (uint32_t t0 = off; t0 < off + seg; t0 += STRETCH) {
        const uint32_t t1 = min(off + seg, t0 + STRETCH);
        if (t0 != off) {
            find_runs<kThreads>(a, seq, kvh, b.lo + 32 * int32_t(t0), b.last, t1 - t0, ms.runs, tid);
            __syncthreads();
        }
        const bool missing = !all_held(ms.runs, t1 - t0, lane_now());

        // ---- tiles into LDS ----
        const uint32_t run_bytes = 16 * rowbytes;
        constexpr int LPR = RB / 16, RPI = 64 / LPR, LOADS = kTileTokens / RPI;  // direct loads of keys or values
        constexpr int MINE = 2 * LOADS / NW;                                   // a wave's
        static_assert(2 * LOADS % NW == 0, "");
        constexpr uint32_t CHUNKS = 2 * kTileTokens * DP / 16;  // 16-byte loads of a tile, 8-bit types
        constexpr int RAW = SCALED ? (CHUNKS + kThreads - 1) / kThreads : 1;  // a thread's
        static_assert(CHUNKS < kThreads || CHUNKS % kThreads == 0, "");
        u32x4 raw[RAW];
        float raw_scale = 0.0f;
        auto load = [&](uint32_t t) __attribute__((always_inline)) {
            const TileRuns w = tile_runs(ms.runs, t - t0);
            const uint32_t buf = (t - t0) % NBUF;
            const uint32_t ln = place_lane();
            if constexpr (!SCALED) {
#pragma unroll
                for (int j = 0; j < MINE; ++j) {
                    const uint32_t f = wave + NW * j;
                    const bool val = LOADS % NW == 0 ? j >= LOADS / NW : f >= uint32_t(LOADS);
                    const uint32_t i = val ? f - LOADS : f, h = i * RPI / 16, rh = i * RPI % 16 + ln / LPR;
                    const uint32_t r = 16 * h + rh;
                    const uint32_t c = (ln % LPR) ^ (val ? value_swizzle<R, RB, 2>(r) : key_swizzle<R, RB>(r));
                    const uint8_t *src = (val ? a.kv.v : a.kv.k) + uint64_t(w.of(h != 0)) * run_bytes;
                    // (dims past the row's: others of it, which meet zeros of q, or go nowhere)
                    dma16((val ? vbuf : kbuf) + buf * TILE + i * 1024, src, rh * rowbytes + (16 * c < rowbytes ? 16 * c : 0));
                }
            } else {
                // 16 bytes (16 dims) of one row per load: kThreads / (DP / 16) rows at a time, keys then values
                const uint32_t tn = 64 * wave + ln;
#pragma unroll
                for (int j = 0; j < RAW; ++j) {
                    const uint32_t f = tn + kThreads * j, c = f % (DP / 16), rr = f / (DP / 16);
                    const bool val = rr >= kTileTokens;
                    const uint32_t r = rr % kTileTokens;
                    const uint8_t *src = (val ? a.kv.v : a.kv.k) + uint64_t(w.of(r >= 16)) * run_bytes + r % 16 * rowbytes;
                    if (CHUNKS >= kThreads || f < CHUNKS) raw[j] = *reinterpret_cast<const u32x4 *>(src + (16 * c < rowbytes ? 16 * c : 0));
                }
                if (wave == 0) raw_scale = (ln >= 32 ? a.kv.vs : a.kv.ks)[16 * uint64_t(w.of(ln & 16)) + ln % 16];
            }
        };
        // (8-bit types) what load() fetched, widened, into its tile
        auto put = [&](uint32_t t) __attribute__((always_inline)) {
            const uint32_t buf = (t - t0) % NBUF, ln = place_lane(), tn = 64 * wave + ln;
#pragma unroll
            for (int j = 0; j < RAW; ++j) {
                const uint32_t f = tn + kThreads * j, c = f % (DP / 16), rr = f / (DP / 16);
                if (CHUNKS < kThreads && f >= CHUNKS) break;
                const bool val = rr >= kTileTokens;
                const uint32_t r = rr % kTileTokens, sw = val ? value_swizzle<R, RB, 2>(r) : key_swizzle<R, RB>(r);
                unsigned char *dst = lds + kMisc + ((val ? NBUF : 0) + buf) * TILE + r * RB;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const u32x2 x = widen<CT>(raw[j][2 * e]), y = widen<CT>(raw[j][2 * e + 1]);
                    *reinterpret_cast<u32x4 *>(dst + (((2 * c + e) ^ sw) << 4)) = u32x4{x[0], x[1], y[0], y[1]};
                }
            }
            if (wave == 0) {
                if (ln < 32) {
                    ms.many.kf[buf][ln] = raw_scale;
                } else {
                    if (__builtin_expect(__ballot(raw_scale == 1.0f) != 0, 0)) {
                        asm volatile("; zeros?");
                        // (from the cache: this tile is on its way to LDS in other waves)
                        const uint8_t *row = a.kv.v + (16 * uint64_t(tile_runs(ms.runs, t - t0).of(ln & 16)) + (ln & 15)) * rowbytes;
                        if (raw_scale == 1.0f && row_of_zeros<CT>(row, rowbytes)) raw_scale = 0.0f;
                    }
                    const float x = value_factor(raw_scale);
                    ms.many.lv[buf][ln - 32] = __builtin_amdgcn_logf(x);
                    ms.many.iv[buf][ln - 32] = __builtin_amdgcn_rcpf(x);
                }
            }
        };

        // whether some row of the wave sees a token of tile t, and whether all see all
        auto any_seen = [&](uint32_t t) {
            const int32_t j0 = b.lo + 32 * int32_t(t);
            return active && j0 <= wlast && int64_t(j0) + 31 + a.span > int64_t(wfirst);
        };
        // Scores as they come from the matrix cores to what the weights are formed
        // from: as they are (times `factor` later), or with a token's factors the
        // exponents of 2 already; unseen ones to -inf; and the largest exponent.
        auto token_factors = [&](uint32_t buf, float (&x)[NS]) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < NS; i += 4) {
                const f32x4 kf = *reinterpret_cast<const f32x4 *>(ms.many.kf[buf] + token_of_reg<R>(i, g));
                const f32x4 lf = *reinterpret_cast<const f32x4 *>(ms.many.lv[buf] + token_of_reg<R>(i, g));
#pragma unroll
                for (int j = 0; j < 4; ++j) x[i + j] = fmaf(x[i + j] * factor, kf[j], lf[j]);
            }
        };
        // (of the lane's own scores: what is above a row's reference shows in one lane)
        auto largest = [&](const float (&x)[NS]) __attribute__((always_inline)) { return SCALED ? max_of(x) : max_of(x) * factor; };
        auto full_tile = [&](uint32_t t) {
            const int32_t j0 = b.lo + 32 * int32_t(t);
            return j0 + 31 <= wfirst && int64_t(j0) + a.span > int64_t(wlast);
        };
        auto finish_scores = [&](uint32_t t, float (&x)[NS]) __attribute__((always_inline)) {
            const int32_t j0 = b.lo + 32 * int32_t(t);
            seen = ALL;
            if constexpr (SCALED) token_factors((t - t0) % NBUF, x);
            if (missing || !full_tile(t)) {
                const uint32_t ok = tile_held(ms.runs, t - t0);
                seen = 0;
                const uint32_t gn = lane_now() / R;
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    const uint32_t tok = token_of_reg<R>(i, gn);
                    const int32_t j = j0 + int32_t(tok);
                    if (j <= pos && j >= from && (ok >> (tok / 16)) & 1) seen |= 1u << i;
                    x[i] = (seen >> i) & 1 ? x[i] : kNegInf;
                }
            }
            tmax = largest(x);
        };
        auto raise = [&]() __attribute__((always_inline)) {
            if (__builtin_expect(__ballot(tmax > m + kLazy) != 0, 0)) {
                asm volatile("; raise");  // (a branch, not 64 products by 1 in every step)
                const float most = groups_max<R>(tmax);
                const float up = most > m + kLazy ? most : m;
                const float al = up == m ? 1.0f : __builtin_amdgcn_exp2f(m - up);
                m = up;
                l *= al;
#pragma unroll
                for (int d = 0; d < DB; ++d) o[d] *= al;
            }
        };
        // the weight of a score
        auto exponential = [&](float x, float ref) __attribute__((always_inline)) {
            return __builtin_amdgcn_exp2f(SCALED ? x - ref : fmaf(x, factor, -ref));
        };

        // ---- the first tiles ----
        load(t0);
        if constexpr (SCALED) put(t0);
        if (t0 + 1 < t1) {
            load(t0 + 1);
            if constexpr (SCALED) put(t0 + 1);
        }
        if (t0 + 2 < t1) load(t0 + 2);
        if constexpr (!SCALED) wait_loads<0>();
        tile_barrier();
        if (any_seen(t0)) {
            products(0, s);
            finish_scores(t0, s);
        }

        // Four tiles at a time, each in its own buffer, so that no address is formed in
        // the loop, as long as every row of the wave sees all of them and the one behind.
        // A tile's score products are issued among the weights of the one before, its
        // value products among the sums and maxima of the one behind, operands
        // AHEAD products ahead of their use. The order is pinned: left to itself the
        // compiler puts the vector work behind the products, and each product right
        // behind its operands.
        auto fast = [&](auto buf_c, uint32_t t, const uint32_t (&kp)[NA], uint32_t vp) __attribute__((always_inline)) {
            constexpr uint32_t buf = decltype(buf_c)::value, nbuf = (buf + 1) % NBUF;
            constexpr int KEYS = NA * KS, VALS = Ge::KT * DB, AHEAD = SHORT ? 2 : 4;
            if constexpr (!SCALED) {
                if (t + 2 < t1)
                    wait_loads<MINE>();
                else
                    wait_loads<0>();
            }
            tile_barrier();
            if constexpr (SCALED)
                if (t + 2 < t1) put(t + 2);
            raise();
            const float ref = (m == kNegInf ? 0.0f : m) - kLift;
            u32x4 op[AHEAD];
            // operand i of the step: keys, then values
            auto operand = [&](int i) __attribute__((always_inline)) {
                if (i < KEYS)
                    op[i % AHEAD] = lds_at((kp[i % NA] ^ key_step<R>(i / NA)) + nbuf * TILE);
                else if (i < KEYS + VALS)
                    op[i % AHEAD] = value_frag<RB>((vp ^ value_block<R>((i - KEYS) % DB)) + buf * TILE, (i - KEYS) / DB);
            };
            Acc<R> y[NA];
#pragma unroll
            for (int i = 0; i < NA; ++i) y[i] = Acc<R>{};
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) operand(i);
            int done = 0;  // weights formed
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < KEYS; ++i) {
#pragma unroll
                for (int p = NP - 1; p >= 0; --p) y[i % NA] = mfma<LT>(op[i % AHEAD], q[p][i / NA], y[i % NA]);
                pin(y[i % NA]);
                operand(i + AHEAD);
#pragma unroll
                for (; done < NS * (i + 1) / KEYS; ++done) s[done] = exponential(s[done], ref);
                if (i == KEYS / 2 && t + 3 < t1) load(t + 3);
                __builtin_amdgcn_sched_barrier(0);
            }
            u32x4 pw[Ge::KT][NP];
            auto pack = [&](int k) __attribute__((always_inline)) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float a = s[8 * k + 2 * j], c = s[8 * k + 2 * j + 1];
#pragma unroll
                    for (int p = 0; p < NP; ++p) pw[k][p][j] = piece2<LT>(a, c);
                }
            };
            float sn[NS], most = kNegInf, sum[2] = {0.0f, 0.0f};
            pack(0);
            int added = 0, compared = 0;
#pragma unroll
            for (int i = 0; i < VALS; ++i) {
                constexpr int half = VALS / 2;
#pragma unroll
                for (int p = NP - 1; p >= 0; --p) o[i % DB] = mfma<LT>(op[(KEYS + i) % AHEAD], pw[i / DB][p], o[i % DB]);
                pin(o[i % DB]);
                operand(KEYS + i + AHEAD);
                if (Ge::KT == 2 && i == 0) pack(1);
#pragma unroll
                for (; added < NS * (i + 1) / VALS; ++added)
                    if constexpr (SCALED)
                        sum[added % 2] = fmaf(s[added], ms.many.iv[buf][token_of_reg<R>(added, g)], sum[added % 2]);
                    else if constexpr (!rounded_sum<CT, NP>())
                        sum[added % 2] += s[added];
                    else if (added % 2 == 1)
                        sum[added / 2 % 2] = add_pair<LT>(pw[added / 8][0][added % 8 / 2], sum[added / 2 % 2]);
                if (i == half) {
#pragma unroll
                    for (int j = 0; j < NS; ++j) sn[j] = y[j / AE][j % AE];
                    if constexpr (SCALED) token_factors(nbuf, sn);
                }
                if (i >= half)
#pragma unroll
                    for (; compared + 2 <= NS * (i - half + 1) / (VALS - half); compared += 2)
                        most = max3(most, sn[compared], sn[compared + 1]);
                __builtin_amdgcn_sched_barrier(0);
            }
            l += sum[0] + sum[1];
            tmax = SCALED ? most : most * factor;
#pragma unroll
            for (int i = 0; i < NS; ++i) s[i] = sn[i];
        };

        for (uint32_t t = t0; t < t1;) {
            if (active && (t - t0) % NBUF == 0 && full_tile(t) && !missing) {
                seen = ALL;
                while (t + 4 < t1 && full_tile(t + 4)) {
                    uint32_t kp[NA];
#pragma unroll
                    for (int i = 0; i < NA; ++i) kp[i] = here(kplace[i]);
                    const uint32_t vp = here(vplace);
                    fast(std::integral_constant<uint32_t, 0>{}, t, kp, vp);
                    fast(std::integral_constant<uint32_t, 1>{}, t + 1, kp, vp);
                    fast(std::integral_constant<uint32_t, 2>{}, t + 2, kp, vp);
                    fast(std::integral_constant<uint32_t, 3>{}, t + 3, kp, vp);
                    t += 4;
                }
            }
            // tile t + 1 is in LDS once every wave is here
            if constexpr (!SCALED) {
                if (t + 2 < t1)
                    wait_loads<MINE>();
                else
                    wait_loads<0>();
            }
            tile_barrier();
            if constexpr (SCALED)
                if (t + 2 < t1) put(t + 2);
            if (t + 3 < t1) load(t + 3);

            const uint32_t buf = (t - t0) % NBUF;
            if (any_seen(t)) {
                raise();
                const float ref = (m == kNegInf ? 0.0f : m) - kLift;
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    s[i] = exponential(s[i], ref);
                    // (the factor of a token that is not seen may be anything)
                    if constexpr (SCALED)
                        l += (seen >> i) & 1 ? s[i] * ms.many.iv[buf][token_of_reg<R>(i, g)] : 0.0f;
                    else if constexpr (!rounded_sum<CT, NP>())
                        l += s[i];
                }
                bool odd = false;  // values that are not finite where some row must not see them
                if (CT != kI8 && __ballot(seen != ALL) != 0) odd = tile_not_finite<LT, TILE>(lds + kMisc + (NBUF + buf) * TILE, lane_now());
                if (!odd) {
                    add_values(buf);
                } else {
                    if constexpr (rounded_sum<CT, NP>())
#pragma unroll
                        for (int i = 0; i < NS; ++i) l += s[i];
                    add_values_one_by_one<LT, R, RB, DP>(lds + kMisc + (NBUF + buf) * TILE, s, seen, lane_now(), o);
                }
            }
            if (t + 1 < t1 && any_seen(t + 1)) {
                products((buf + 1) % NBUF, s);
                finish_scores(t + 1, s);
            }
            ++t;
        }
        __syncthreads();  // (the stretch's runs are no longer read)
        }

        // ---- the sums ----
        l = groups_sum<R>(l);
        const uint32_t gn = lane_now() / R;
        const bool whole = off == 0 && seg == b.tiles;
        const uint32_t slot = 2 * work.id + (first_seg ? 0 : 1);
        if (row < b.rows) {
            if (whole) {
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int k = 0; k < AE / 4; ++k) {
                        const uint32_t e = R * d + dim_of_quad(k, gn);
                        const f32x4 x = {o[d][4 * k], o[d][4 * k + 1], o[d][4 * k + 2], o[d][4 * k + 3]};
                        if (e < D) store4(a, b.begin, kvh, row, e, x * inv);
                    }
            } else {
                const uint64_t at = uint64_t(slot) * SLOT + row - r0;
                if (gn == 0) sc.ml[2 * at] = m, sc.ml[2 * at + 1] = l;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int k = 0; k < AE / 4; ++k)
                        *reinterpret_cast<f32x4 *>(sc.o + at * DP + R * d + dim_of_quad(k, gn)) =
                            f32x4{o[d][4 * k], o[d][4 * k + 1], o[d][4 * k + 2], o[d][4 * k + 3]};
            }
        }
        // this workgroup has the block's first tiles but not its last: the join is on its list
        if (off == 0 && !whole && tid == 0)
            sc.jobs[work.id] = SplitJob{b.begin, r0, kvh, min(uint32_t(Sh::ROWS), b.rows - r0), 1 + uint32_t((b.tiles - seg + work.part - 1) / work.part), slot};
        left -= sg.places;
        first_seg = false;
        if (left != 0 && !next_block<Sh::ROWS>(a, rg, seqs, b.rows, pl)) break;
    }
}

}  // namespace
}  // namespace tc
