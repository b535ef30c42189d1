// tc_rope.hip -- rotary positions, on rows and on the way into a paged cache.
//
// A pair (u, v) of a head becomes m (u cos a - v sin a, u sin a + v cos a) with a = 2 pi p
// turns_i. The product p * turns_i is formed in fp64 and its whole turns are taken off there:
// 53 bits leave 2^-24 of a turn at positions near 2^31, where an fp32 angle would be off
// by whole turns (at 10^5 by 2^-7 radians). What is left of a turn, less the nearest
// quarter, is at most an eighth, and sin and cos of it are their Taylor series in fp32.
//
// A lane has 8 consecutive dims of `U` heads of one token, whose angles it forms once; the
// other halves of its pairs are in the same 8 dims (TC_ROPE_PAIRS) or are read a second time
// from the row (TC_ROPE_HALF: out of L1, the row is loaded by the neighbouring lanes at the
// same time). So each row goes from HBM to HBM once, and both kernels are bound by that for
// prompts, and by the chain start -> len -> table -> store for single tokens.
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
    DivMod groups;      // of U units in a token
    uint32_t total;     // groups of all tokens
};

// The 8 factors of a lane's dims from `at` on: out[i] = x[i] * c[i] + other[i] * s[i].
__device__ __forceinline__ void angles(const RopeArgs &r, uint32_t at, int32_t pos, float (&c)[8], float (&s)[8]) {
    const double p = double(pos);
    if (r.layout == TC_ROPE_PAIRS) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t e = at + 2 * i;
            float cs = 1.0f, sn = 0.0f;
            if (e < r.n_rot) {
                turn(p * r.turns[e >> 1], &cs, &sn);
                cs *= r.factor, sn *= r.factor;
            }
            c[2 * i] = c[2 * i + 1] = cs;
            s[2 * i] = -sn, s[2 * i + 1] = sn;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t e = at + i;
            const bool second = e >= r.half;
            c[i] = 1.0f, s[i] = 0.0f;
            if (e < r.n_rot) {
                turn(p * r.turns[second ? e - r.half : e], &c[i], &s[i]);
                c[i] *= r.factor, s[i] *= second ? r.factor : -r.factor;
            }
        }
    }
}

__device__ __forceinline__ float load1(int type, const void *p, uint64_t elem) {
    if (type == kF32) return static_cast<const float *>(p)[elem];
    const uint32_t w = static_cast<const uint16_t *>(p)[elem];
    return type == kF16 ? h2f(w) : __builtin_bit_cast(float, w << 16);
}

// The other halves of the pairs of the row's dims from `at` on (whatever it is where there
// is none).
__device__ __forceinline__ void load_others(const RopeArgs &r, int type, const void *p, uint64_t row, uint32_t at,
                                            const float (&x)[8], float (&y)[8]) {
    if (r.layout == TC_ROPE_PAIRS) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = x[i ^ 1];
    } else if ((r.half & 7) == 0) {
        const uint32_t e = at < r.half ? at + r.half : at < r.n_rot ? at - r.half : at;
        load8(type, p, row + e, y);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t e = at + i, o = e < r.half ? e + r.half : e < r.n_rot ? e - r.half : e;
            y[i] = load1(type, p, row + o);
        }
    }
}
__device__ __forceinline__ float weight_of(const RopeArgs &r, const float *w, uint32_t e) {
    if (r.layout == TC_ROPE_PAIRS) return w[e ^ 1];
    return w[e < r.half ? e + r.half : e < r.n_rot ? e - r.half : e];
}

// CT: the cache's type, kF32 where there is none (positions are given, all units are q's).
template <int CT, int U>
__global__ __launch_bounds__(kThreads) void k_rope(RopeCall a, RopeWalk w) {
    constexpr bool CACHE = CT != kF32;
    const uint32_t dim = a.kv.dim;
    const uint32_t g = (blockIdx.x << (8 - w.lane_log)) + (threadIdx.x >> w.lane_log);
    const uint32_t at = (threadIdx.x & (w.lanes - 1)) * 8;
    // lanes without work go through it all the same (the rows' lanes agree on sums and
    // maxima), on the last row, and store nothing
    const uint32_t gc = min(g, w.total - 1), t = div_fast(gc, w.groups), u0 = (gc - t * w.groups.d) * U;
    const bool mine = g < w.total && at < dim;
    const uint32_t from = at < dim ? at : 0;
    float x[U][8], y[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t n = min(u0 + u, w.units - 1);
        const bool is_q = !CACHE || n < a.q.heads, is_k = CACHE && !is_q && n - a.q.heads < a.k.heads;
        const uint32_t h = is_q ? n : is_k ? n - a.q.heads : n - a.q.heads - a.k.heads;
        const RopeHeads &src = is_q ? a.q : is_k ? a.k : a.v;
        const uint64_t row = uint64_t(t) * src.stride + h * dim;
        load8(a.xtype, src.x, row + from, x[u]);
        if (is_q || is_k) load_others(a.rope, a.xtype, src.x, row, from, x[u], y[u]);
        if (at >= dim)  // (of a row's largest magnitude and sum of squares these lanes have nothing)
#pragma unroll
            for (int i = 0; i < 8; ++i) x[u][i] = y[u][i] = 0.0f;
    }
    int32_t pos;
    int seq = 0;
    int64_t row0 = -1;  // cache row of head 0
    if constexpr (CACHE) {
        const uint32_t first = min(div_fast(min(blockIdx.x << (8 - w.lane_log), w.total - 1), w.groups), a.kv.n_tokens - 1);
        seq = wave_find_seq(a.kv.start, a.kv.n_seq, first);
        const int32_t end = seq >= 0 ? a.kv.start[seq + 1] : 0;
        if (int32_t(t) >= end) seq = find_seq(a.kv.start, a.kv.n_seq, t);
        const uint32_t s = seq < 0 ? 0 : uint32_t(seq);
        pos = int32_t(int64_t(a.kv.len[s]) - a.kv.start[s + 1] + t);
        row0 = slot_of(a.kv, seq, t, 0);
    } else {
        pos = a.position[t];
        if (pos < 0) seq = -1;
    }
    float c[8], s[8];
    if (!CACHE || u0 < a.q.heads + a.k.heads) angles(a.rope, from, pos, c, s);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t n = u0 + u;
        const bool is_q = !CACHE || n < a.q.heads, is_k = CACHE && !is_q && n - a.q.heads < a.k.heads;
        const bool live = mine && n < w.units && seq >= 0;
        if (is_q || is_k) {
            if constexpr (CACHE) {
                const float *nw = is_q ? a.q.norm : a.k.norm;
                if (nw != nullptr) {  // uniform over the row's lanes, which have the same unit
                    float m = 0.0f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) m = __builtin_fmaf(x[u][i], x[u][i], m);
                    for (uint32_t o = 1; o < w.lanes; o <<= 1) m += __shfl_xor(m, int(o));
                    const float inv = rsqrtf(m / float(dim) + a.eps);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        x[u][i] = x[u][i] * inv * nw[from + i];
                        y[u][i] = y[u][i] * inv * weight_of(a.rope, nw, from + i);
                    }
                }
            }
            float o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                o[i] = at + i < a.rope.n_rot ? __builtin_fmaf(x[u][i], c[i], y[u][i] * s[i]) : x[u][i];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[u][i] = o[i];
            if (is_q) {
                if (live) store8(a.xtype, a.q_out, uint64_t(t) * a.q_out_stride + n * dim + at, x[u]);
                continue;
            }
        }
        if constexpr (CACHE) {
            const uint32_t h = is_k ? n - a.q.heads : n - a.q.heads - a.k.heads;
            put_row<CT>(is_k ? a.kv.k : a.kv.v, is_k ? a.kv.ks : a.kv.vs, dim,
                        row0 < 0 ? -1 : row0 + int64_t(h) * a.kv.page, at, live, w.lanes, x[u]);
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
    w.lanes = 2, w.lane_log = 1;
    while (w.lanes * 8 < c.kv.dim) w.lanes *= 2, ++w.lane_log;
    w.units = units;
    const uint32_t groups = (units + per_lane - 1) / per_lane;
    w.groups = make_divmod(groups);
    w.total = c.kv.n_tokens * groups;
    const uint32_t rows = kThreads / w.lanes;
    *blocks = (w.total + rows - 1) / rows;
    return w;
}

template <int CT>
hipError_t launch(const RopeCall &c, uint32_t units, hipStream_t st) {
    uint32_t blocks;
    RopeWalk w = make_walk(c, units, 1, &blocks);
    if (blocks <= 4096) {
        k_rope<CT, 1><<<blocks, kThreads, 0, st>>>(c, w);
    } else {
        w = make_walk(c, units, 4, &blocks);
        k_rope<CT, 4><<<blocks, kThreads, 0, st>>>(c, w);
    }
    return hipGetLastError();
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
