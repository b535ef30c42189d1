// tc_rope.hip -- rotary positions, on rows and on the way into a paged cache.
//
// A pair (u, v) of a head becomes m (u cos a - v sin a, u sin a + v cos a) with a = 2 pi p
// turns_i. The product p * turns_i is formed in fp64 and its whole turns are taken off there:
// 53 bits leave 2^-24 of a turn at positions near 2^31, where an fp32 angle would be off
// by whole turns (at 10^5 by 2^-7 radians). What is left of a turn, less the nearest
// quarter, is at most an eighth, and sin and cos of it are their Taylor series in fp32.
//
// A lane has 8 consecutive dims of one or four heads of a token, whose angles it forms once; the
// other halves of its pairs are in the same 8 dims (TC_ROPE_PAIRS) or are read a second time
// from the row (TC_ROPE_HALF: out of L1, the row is loaded by the neighbouring lanes at the
// same time). So each row goes from HBM to HBM once: prompts are bound by that (8190 rows of 36
// heads of 128, bf16: 30 us, 151 MB at 5.0 TB/s; VALU 0.56 busy, half of it the angles and addresses
// of a wave that does nothing twice), single tokens by the chain start -> len -> table -> store (3.5
// us; 241 rows with norms and 8-bit values 5.9 to 6.2).
// That prompt is of pairs, half of each head. All of it rotated, pairs take 32 us, halves 35, since both lanes of
// their pairs form the angles and load both values; with norms of heads 36 and 44; halves of n_rot / 2 = 61, whose
// partners are loaded one by one, 48.
//
// Not kept: the same heads of several tokens in a wave, which makes the choice between q, k and v a
// scalar's (38 us for 37, and 6.9 for 6.2: a wave's tokens are of several sequences), two, eight
// or twelve heads a lane (36, 36, 37 for 34).
#include "tc_kernels.hpp"
#include "tc_kv_put.hpp"
#include "tc_step.hpp"

namespace tc {
namespace {

constexpr uint32_t kThreads = 256;

// cos and sin of 2 pi p turns, for |p turns| up to 2^52.
__device__ __forceinline__ void turn(double t, float *c, float *s) {
    const double q = __builtin_rint(4.0 * t);                    // quarters
    const float x = float(__builtin_fma(q, -0.25, t) * 6.283185307179586);  // in [-pi/4, pi/4]
    const float z = x * x;
    // x - x^3/3! + .. + x^9/9!, 1 - x^2/2! + .. + x^8/8!: the terms left out are below
    // 2^-29 and 2^-25
    float sn = __builtin_fmaf(z, 2.75573192e-6f, -1.98412698e-4f);
    sn = __builtin_fmaf(z, sn, 8.33333333e-3f);
    sn = __builtin_fmaf(z, sn, -1.66666667e-1f);
    sn = __builtin_fmaf(x * z, sn, x);
    float cs = __builtin_fmaf(z, 2.48015873e-5f, -1.38888889e-3f);
    cs = __builtin_fmaf(z, cs, 4.16666667e-2f);
    cs = __builtin_fmaf(z, cs, -0.5f);
    cs = __builtin_fmaf(z, cs, 1.0f);
    // the quarter's number, modulo 4, out of the low bits of the sum with 1.5 * 2^52
    const uint32_t n = uint32_t(__builtin_bit_cast(uint64_t, q + 6755399441055744.0));
    const float a = n & 1 ? sn : cs, b = n & 1 ? cs : sn;
    *c = (n + 1) & 2 ? -a : a;
    *s = n & 2 ? -b : b;
}

// How a launch goes over the units: heads of a token's q, k and v, one after the other; U
// of them are a lane's.
struct RopeWalk {
    uint32_t lanes;     // of a head, a power of two
    uint32_t lane_log;  // its logarithm
    uint32_t units;     // of a token
    DivMod groups;      // of U units in a token, that many units apart
    uint32_t total;     // groups of all tokens
};

// How a head's dims pair up: neighbours; halves of 8's multiples, so that the other halves of a
// lane's pairs are one load; any halves.
enum : int { kPairs, kHalves8, kHalves };

// The turns of the pairs of a lane's dims from `at` on (kPairs: of its 4 pairs).
template <int L>
__device__ __forceinline__ void load_turns(const RopeArgs &r, uint32_t at, double (&t)[8]) {
#pragma unroll
    for (int i = 0; i < (L == kPairs ? 4 : 8); ++i) {
        const uint32_t e = L == kPairs ? at / 2 + i : at + i;
        t[i] = r.turns[min(L == kPairs || e < r.half ? e : e - r.half, r.half - 1)];
    }
}
// The factors of those dims at a position: out[i] = x[i] * c[i] + other[i] * s[i].
template <int L>
__device__ __forceinline__ void angles(const RopeArgs &r, uint32_t at, int32_t pos, const double (&t)[8], float (&c)[8], float (&s)[8]) {
    const double p = double(pos);
    if constexpr (L == kPairs) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float cs, sn;
            turn(p * t[i], &cs, &sn);
            c[2 * i] = c[2 * i + 1] = cs * r.factor;
            s[2 * i + 1] = sn * r.factor, s[2 * i] = -s[2 * i + 1];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            turn(p * t[i], &c[i], &s[i]);
            c[i] *= r.factor, s[i] *= at + i < r.half ? -r.factor : r.factor;
        }
    }
}

// 8 values as they are in memory. W: an element's bytes.
template <int W>
struct Raw {
    u32x4 v[W / 2];
};
template <int W>
__device__ __forceinline__ Raw<W> raw_load(const void *p, uint64_t elem) {
    Raw<W> r;
    const u32x4 *q = reinterpret_cast<const u32x4 *>(static_cast<const uint8_t *>(p) + elem * W);
    r.v[0] = q[0];
    if constexpr (W == 4) r.v[1] = q[1];
    return r;
}
template <int W>
__device__ __forceinline__ void widen(int type, const Raw<W> &r, float (&x)[8]) {
    if constexpr (W == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __builtin_bit_cast(float, uint32_t(r.v[i / 4][i & 3]));
    } else if (type == kF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[2 * i] = h2f(r.v[0][i] & 0xFFFF), x[2 * i + 1] = h2f(r.v[0][i] >> 16);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __builtin_bit_cast(float, uint32_t(r.v[0][i]) << 16);
            x[2 * i + 1] = __builtin_bit_cast(float, r.v[0][i] & 0xFFFF0000u);
        }
    }
}

// The dim that dim e is a pair with; e itself behind the rotated ones.
template <int L>
__device__ __forceinline__ uint32_t other_of(const RopeArgs &r, uint32_t e) {
    if constexpr (L == kPairs) return e ^ 1;
    return e < r.half ? e + r.half : e < r.n_rot ? e - r.half : e;
}

// A norm's weights for 8 dims from `at` on, and for those that they are pairs with.
typedef float f32x4d __attribute__((ext_vector_type(4), aligned(4)));
template <int L>
__device__ __forceinline__ void load_norm(const RopeArgs &r, const float *n, uint32_t at, float (&w)[8], float (&o)[8]) {
    auto load = [&](uint32_t from, float (&x)[8]) {
        const f32x4d *q = reinterpret_cast<const f32x4d *>(n + from);
        const f32x4d u = q[0], v = q[1];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = u[i], x[4 + i] = v[i];
    };
    load(at, w);
    if constexpr (L == kPairs) {
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = w[i ^ 1];
    } else if constexpr (L == kHalves8) {
        load(other_of<L>(r, at), o);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = n[other_of<L>(r, at + i)];
    }
}

// CT: the cache's type, kF32 where there is none (positions are given, all units are q's). W:
// bytes of the rows' elements. L: layout. U: units of a lane.
template <int CT, int W, int L, int U>
__global__ __launch_bounds__(kThreads) void k_rope(RopeCall a, RopeWalk w) {
    constexpr bool CACHE = CT != kF32;
    const uint32_t dim = a.kv.dim;
    const uint32_t g = (blockIdx.x << (8 - w.lane_log)) + (threadIdx.x >> w.lane_log);
    const uint32_t at = (threadIdx.x & (w.lanes - 1)) * 8;
    // lanes without work go through it all the same (the rows' lanes agree on sums and
    // maxima), on the last row, and store nothing
    const uint32_t gc = min(g, w.total - 1), t = div_fast(gc, w.groups), u0 = gc - t * w.groups.d;
    const bool mine = g < w.total && at < dim;
    const uint32_t from = at < dim ? at : 0;
    // (all loads first, and without branches between them: each would wait for the one before;
    // what others depend on in front)
    const uint32_t first = min(div_fast(min(blockIdx.x << (8 - w.lane_log), w.total - 1), w.groups), a.kv.n_tokens - 1);
    SeqProbe probe;
    if constexpr (CACHE) probe = probe_seqs(a.kv.start, a.kv.n_seq);
    Raw<W> x_raw[U], y_raw[U];
    uint64_t row[U];
    const void *src[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t n = min(u0 + u * w.groups.d, w.units - 1);
        const bool is_q = !CACHE || n < a.q.heads, is_k = CACHE && !is_q && n - a.q.heads < a.k.heads;
        const uint32_t h = is_q ? n : is_k ? n - a.q.heads : n - a.q.heads - a.k.heads;
        src[u] = is_q ? a.q.x : is_k ? a.k.x : a.v.x;
        row[u] = uint64_t(t) * (is_q ? a.q.stride : is_k ? a.k.stride : a.v.stride) + h * dim;
        x_raw[u] = raw_load<W>(src[u], row[u] + from);
        if constexpr (L == kHalves8) y_raw[u] = raw_load<W>(src[u], row[u] + other_of<L>(a.rope, from));
    }
    // (the heads' weights of a single unit too, which wait for nothing)
    float nw[8], no[8];
    bool normed = false;
    if constexpr (CACHE && U == 1) {
        const float *n = u0 < a.q.heads ? a.q.norm : u0 - a.q.heads < a.k.heads ? a.k.norm : nullptr;
        normed = n != nullptr;
        if (normed) load_norm<L>(a.rope, n, from, nw, no);
    }
    // (long calls have the turns on their way from here, 39 -> 35 us for 8190 rows; short ones'
    // lookups would wait for them, 6.0 -> 6.7 for 241)
    double turns[8];
    if constexpr (U > 1) load_turns<L>(a.rope, from, turns);
    int32_t pos;
    int seq = 0;
    int64_t row0 = -1;  // cache row of head 0
    if constexpr (CACHE) {
        seq = wave_find_seq(a.kv.start, a.kv.n_seq, first, probe);
        const uint32_t s0 = seq < 0 ? 0 : uint32_t(seq);
        int32_t end = a.kv.start[s0 + 1], len = a.kv.len[s0];
        if (seq < 0 || int32_t(t) >= end) {
            seq = find_seq(a.kv.start, a.kv.n_seq, t);
            if (seq >= 0) end = a.kv.start[seq + 1], len = a.kv.len[seq];
        }
        const int64_t at = int64_t(len) - end + t;
        pos = int32_t(at);
        if (seq >= 0 && at >= 0 && at < int64_t(kMaxPos)) {
            const uint32_t pi = div_fast(uint32_t(pos), a.kv.page_div);
            const int32_t page = page_at(a.kv, uint32_t(seq), pi);
            if (page >= 0) row0 = int64_t(page) * a.kv.kv_heads * a.kv.page + (uint32_t(pos) - pi * a.kv.page);
        }
    } else {
        pos = a.position[t];
        if (pos < 0) seq = -1;
    }
    if constexpr (U == 1) load_turns<L>(a.rope, from, turns);
    float c[8], s[8];
    if (!CACHE || u0 < a.q.heads + a.k.heads) angles<L>(a.rope, from, pos, turns, c, s);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t n = u0 + u * w.groups.d;
        const bool is_q = !CACHE || n < a.q.heads, is_k = CACHE && !is_q && n - a.q.heads < a.k.heads;
        const bool live = mine && n < w.units && seq >= 0;
        float x[8], y[8];
        widen<W>(a.xtype, x_raw[u], x);
        if (at >= dim)  // (of a row's largest magnitude and sum of squares these lanes have nothing)
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = 0.0f;
        if (is_q || is_k) {
            if constexpr (L == kPairs) {
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = x[i ^ 1];
            } else if constexpr (L == kHalves8) {
                widen<W>(a.xtype, y_raw[u], y);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint64_t e = row[u] + other_of<L>(a.rope, from + i);
                    if constexpr (W == 4) {
                        y[i] = static_cast<const float *>(src[u])[e];
                    } else {
                        const uint32_t bits = static_cast<const uint16_t *>(src[u])[e];
                        y[i] = a.xtype == kF16 ? h2f(bits) : __builtin_bit_cast(float, bits << 16);
                    }
                }
            }
            if constexpr (CACHE) {
                if constexpr (U > 1) {
                    const float *n = is_q ? a.q.norm : a.k.norm;
                    normed = n != nullptr;
                    if (normed) load_norm<L>(a.rope, n, from, nw, no);
                }
                if (normed) {  // all of the row's lanes, which have the same unit
                    float m = 0.0f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) m = __builtin_fmaf(x[i], x[i], m);
                    const float inv = rsqrtf(group_sum(m, w.lanes) / float(dim) + a.eps);
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * nw[i], y[i] = y[i] * inv * no[i];
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = at + i < a.rope.n_rot ? __builtin_fmaf(x[i], c[i], y[i] * s[i]) : x[i];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = y[i];
            if (is_q) {
                if (live) store8(a.xtype, a.q_out, uint64_t(t) * a.q_out_stride + n * dim + at, x);
                continue;
            }
        }
        if constexpr (CACHE) {
            const uint32_t h = is_k ? n - a.q.heads : n - a.q.heads - a.k.heads;
            put_row<CT>(is_k ? a.kv.k : a.kv.v, is_k ? a.kv.ks : a.kv.vs, dim,
                        row0 < 0 ? -1 : row0 + int64_t(h) * a.kv.page, at, live, w.lanes, x);
        }
    }
}

__global__ __launch_bounds__(64) void k_rope_turns(TurnsCall a) {
    const uint32_t i = blockIdx.x * 64 + threadIdx.x;
    if (i >= a.n_rot / 2) return;
    const double n = a.n_rot, whole = 0.15915494309189535;  // 1 / (2 pi)
    double theta = a.theta;
    if (a.kind == TC_ROPE_NTK) theta *= pow(a.factor, n / (n - 2.0));
    double t = pow(theta, -2.0 * i / n) * whole, part = 0.0;  // part: how far f_i goes to f_i / s
    if (a.kind == TC_ROPE_LINEAR) part = 1.0;
    if (a.kind == TC_ROPE_YARN) part = (i - a.first) / a.ramp;
    if (a.kind == TC_ROPE_BANDS) part = 1.0 - (a.original * t - a.low) / (a.high - a.low);
    part = fmin(fmax(part, 0.0), 1.0);
    t = t * (1.0 - part) + t / a.factor * part;
    a.turns[i] = a.divisors != nullptr ? t / double(a.divisors[i]) : t;
}

RopeWalk make_walk(const RopeCall &c, uint32_t units, uint32_t per_lane, uint32_t *blocks) {
    RopeWalk w;
    w.lane_log = rope_lane_log(c.kv.dim);
    w.lanes = 1u << w.lane_log;
    w.units = units;
    const uint32_t groups = (units + per_lane - 1) / per_lane;
    w.groups = make_divmod(groups);
    w.total = c.kv.n_tokens * groups;
    const uint32_t rows = kThreads / w.lanes;
    *blocks = (w.total + rows - 1) / rows;
    return w;
}

template <int CT, int W, int L>
hipError_t launch(const RopeCall &c, uint32_t units, hipStream_t st) {
    uint32_t blocks;
    RopeWalk w = make_walk(c, units, 1, &blocks);
    // (four heads a lane from where single ones are more than 4 workgroups per CU. Rows and cache of 16
    // bits, 28 + 2 x 4 heads of 128, us with one and with four: halves, 8190 rows 61 and 35, 1024 10.4 and 8.6,
    // 512 6.4 and 6.5, 256 5.1 and 5.4; pairs 42.5 and 32.5, 7.9 and 7.1, 5.3 and 5.4, 4.2 and 4.8; halves with
    // norms of heads 66 and 44, 11.2 and 9.7, 6.9 and 7.4, 5.3 and 6.1)
    if (blocks <= 1024) {
        k_rope<CT, W, L, 1><<<blocks, kThreads, 0, st>>>(c, w);
    } else {
        w = make_walk(c, units, kRopeUnits, &blocks);
        k_rope<CT, W, L, kRopeUnits><<<blocks, kThreads, 0, st>>>(c, w);
    }
    return hipGetLastError();
}
template <int CT, int W>
hipError_t launch(const RopeCall &c, uint32_t units, hipStream_t st) {
    if (c.rope.layout == TC_ROPE_PAIRS) return launch<CT, W, kPairs>(c, units, st);
    return c.rope.half % 8 == 0 ? launch<CT, W, kHalves8>(c, units, st) : launch<CT, W, kHalves>(c, units, st);
}
template <int CT>
hipError_t launch(const RopeCall &c, uint32_t units, hipStream_t st) {
    return c.xtype == kF32 ? launch<CT, 4>(c, units, st) : launch<CT, 2>(c, units, st);
}

}  // namespace

hipError_t launch_rope_kv(const RopeCall &c, int ctype, hipStream_t st) {
    const uint32_t units = c.q.heads + 2 * c.k.heads;
    switch (ctype) {
        case kF16: return launch<kF16>(c, units, st);
        case kBF16: return launch<kBF16>(c, units, st);
        case kI8: return launch<kI8>(c, units, st);
        default: return launch<kE4M3>(c, units, st);
    }
}

hipError_t launch_rope_rows(const RopeCall &c, hipStream_t st) { return launch<kF32>(c, c.q.heads, st); }

hipError_t launch_rope_turns(const TurnsCall &c, hipStream_t st) {
    k_rope_turns<<<(c.n_rot / 2 + 63) / 64, 64, 0, st>>>(c);
    return hipGetLastError();
}

}  // namespace tc
