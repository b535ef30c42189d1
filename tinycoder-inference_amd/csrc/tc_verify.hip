// tc_verify.hip -- verification of drafted tokens against the target's logits.
//
// Three launches. k_verify_rows reads every logit once: for a slice of a row the
// largest and the sum of exponentials (where the temperature is 0: the largest and its
// lowest index). k_verify_weights joins a sequence's slices, walks its drafts, and sums
// the sampling weights of the row where they end, again in slices; k_verify_pick finds
// the slice and then the token that the random number falls on. The first takes 39 to 44 us
// for 263 rows of 152064 logits (160 MB at 3.6 to 4.1 TB/s; VALU busy for two thirds of
// that time, with fp64), the others 19 to 24 and 7 to 8 us for their 48 sequences (each of
// the second's workgroups walks its sequence's drafts before it reads 53 MB in all).
//
// Everything behind the logits is fp64: a token's probability in a vocabulary of
// 10^5 is 10^-5 and less, so sums in fp32 would move the borders between tokens by
// a hundredth of their width.
#include <algorithm>

#include "tc_attn_common.hpp"
#include "tc_kernels.hpp"

namespace tc {
namespace {

constexpr uint32_t kThreads = 256;      // of k_verify_rows
constexpr uint32_t kThreadsSeq = 512;   // of k_verify_weights
constexpr uint32_t kThreadsPick = 256;  // of k_verify_pick
constexpr float kInf = __builtin_inff();

// (4-byte aligned: rows of an odd vocabulary)
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

// A slice of a row: its largest logit, the sum of exp((l - m) / temperature), and at
// temperature 0 that logit's lowest index instead. A NaN among the logits gives a NaN sum.
struct Slice {
    double sum;
    float m;
    int32_t at;
};
// A slice's sampling weights: of the residual, and of p alone.
struct Weight {
    double rest, full;
};
// Where a sequence's drafts ended.
struct Stop {
    double inv;      // 1 / sum of the row's exponentials
    float m;         // its largest logit
    int32_t row;     // -1: no row
    int32_t draft;   // the rejected draft, -1 where none was
    int32_t good;    // the row can be sampled from
};

struct Split {
    uint32_t rows_n, rows_len, pick_n, pick_len;  // slices and their lengths, both kernels
};

__host__ __device__ inline uint32_t div_up(uint32_t a, uint32_t b) { return (a + b - 1) / b; }

// As many slices as make about kRowsPerCu workgroups per CU, of 2048 logits or more (8 of
// a thread); and kPickPerCu waves, of 512 or more (as many as the card holds at a time, for
// each workgroup walks the drafts: 48 sequences of 263 rows 70 us in all, 74 with 32 waves).
constexpr uint32_t kRowsPerCu = 16, kPickPerCu = 24;
constexpr int kMostCu = 256;
Split split(uint32_t vocab, uint32_t n_tokens, uint32_t n_seq, int num_cu) {
    auto length = [&](uint32_t want, uint32_t rows, uint32_t least) {
        const uint32_t n = std::min(std::max(want / rows, 1u), div_up(vocab, least));
        return div_up(div_up(vocab, n), 4) * 4;
    };
    Split s;
    s.rows_len = length(kRowsPerCu * uint32_t(num_cu), n_tokens, 2048);
    s.rows_n = div_up(vocab, s.rows_len);
    s.pick_len = length(kPickPerCu * uint32_t(num_cu), n_seq, 512);
    s.pick_n = div_up(vocab, s.pick_len);
    return s;
}

// What stands N lanes to the left and the like (DPP); 0 where there is none.
template <int CTRL, int ROWS>
__device__ __forceinline__ double other_lane(double v) {
    const uint64_t x = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, int(uint32_t(x)), CTRL, ROWS, 15, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, int(uint32_t(x >> 32)), CTRL, ROWS, 15, false);
    return __builtin_bit_cast(double, uint64_t(hi) << 32 | lo);
}
__device__ __forceinline__ double lane_value(double v, uint32_t lane) {
    const uint64_t x = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane(uint32_t(x), lane), hi = __builtin_amdgcn_readlane(uint32_t(x >> 32), lane);
    return __builtin_bit_cast(double, uint64_t(hi) << 32 | lo);
}
// The wave's sums up to each lane, and its sum. All lanes call them.
__device__ __forceinline__ double wave_scan(double v) {
    v += other_lane<0x111, 15>(v);  // 1, 2, 4, 8 lanes to the left in rows of 16
    v += other_lane<0x112, 15>(v);
    v += other_lane<0x114, 15>(v);
    v += other_lane<0x118, 15>(v);
    v += other_lane<0x142, 10>(v);  // the last lane of rows 0 and 2 to rows 1 and 3
    v += other_lane<0x143, 12>(v);  // lane 31 to rows 2 and 3
    return v;
}
__device__ __forceinline__ double wave_sum(double v) { return lane_value(wave_scan(v), 63); }

// log2(e) / temperature, 0 for the greedy choice; and the difference of logits below
// which a token's share is taken for 0 (2^-900). An infinite temperature's factor is not 0:
// with 1e-60 a difference of finite logits, up to 2^129, is nothing, and -inf still below
// every difference.
struct Scale {
    double c, least;
};
__device__ __forceinline__ Scale scale_of(float t) {
    if (!(t > 0.0f)) return Scale{0.0, 0.0};
    const double c = __builtin_fmax(1.4426950408889634 / double(t), 1e-60);
    return Scale{c, -900.0 / c};
}

// 2^(d * c) for least <= d <= 900 / c. The whole part n of the exponent stands in the low
// bits of a sum with 1.5 * 2^52 and goes into the result's exponent field; 2^f for the rest,
// in [-1/2, 1/2], is the polynomial of degree 10 through its values at the 11 Chebyshev
// nodes there: its error is 3e-16 of the value, two roundings' (degree 9: 2e-14), and
// 2^0 is 1. A third of the library function's instructions, which took more time than the
// logits' way from HBM (263 rows of 152064 logits 88 us).
__device__ __forceinline__ double power(double d, double c) {
    constexpr double kShift = 6755399441055744.0;
    const double k = __builtin_fma(d, c, kShift), f = __builtin_fma(d, c, kShift - k);
    double y = 7.072585949269224e-09;
    y = __builtin_fma(y, f, 1.0208690299958306e-07);
    y = __builtin_fma(y, f, 1.321544258792169e-06);
    y = __builtin_fma(y, f, 1.5252657260200837e-05);
    y = __builtin_fma(y, f, 0.0001540353044173605);
    y = __builtin_fma(y, f, 0.0013333558230164974);
    y = __builtin_fma(y, f, 0.009618129107606888);
    y = __builtin_fma(y, f, 0.05550410866444772);
    y = __builtin_fma(y, f, 0.24022650695910097);
    y = __builtin_fma(y, f, 0.69314718055995);
    y = __builtin_fma(y, f, 1.0);
    const uint64_t b = __builtin_bit_cast(uint64_t, y), n = __builtin_bit_cast(uint64_t, k);
    return __builtin_bit_cast(double, b + (n << 52));
}
// The share of a logit x beside m >= x; 0 for -inf and NaN.
__device__ __forceinline__ double share(float x, float m, Scale z) {
    const double d = double(x) - double(m);
    const double y = power(__builtin_fmax(d, z.least), z.c);
    return d > z.least ? y : 0.0;
}

// (m, at) of the larger logit, the lower index where they are alike.
__device__ __forceinline__ void take_larger(float &m, int32_t &at, float om, int32_t oat) {
    if (om > m || (om == m && oat < at)) m = om, at = oat;
}

// Four entries of a row from i on, `pad` from the slice's end on.
__device__ __forceinline__ void four(const float *l, uint32_t i, uint32_t i1, float pad, float *x) {
    if (i + 4 <= i1) {
        const f32x4u v = *reinterpret_cast<const f32x4u *>(l + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = v[j];
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = i + j < i1 ? l[i + j] : pad;
    }
}

__global__ __launch_bounds__(kThreads) void k_verify_rows(VerifyArgs a, Split sp, Slice *__restrict__ out) {
    constexpr uint32_t W = kThreads / 64;
    const uint32_t t = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int s = wave_find_seq(a.start, a.n_seq, t);
    if (s < 0) return;
    const Scale z = scale_of(a.temperature[s]);
    const float *l = a.logits + size_t(t) * a.vocab;
    const uint32_t i0 = blockIdx.x * sp.rows_len, i1 = min(i0 + sp.rows_len, a.vocab);
    __shared__ float sm[W];
    __shared__ int32_t sa[W];
    __shared__ double ss[W];
    float m = -kInf;  // the largest; NaN stays
    if (z.c == 0.0) {
        float best = -kInf;
        int32_t at = 0x7FFFFFFF;
        for (uint32_t i = i0 + 4 * threadIdx.x; i < i1; i += 4 * kThreads) {
            float x[4];
            four(l, i, i1, -kInf, x);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                m = __builtin_elementwise_maximum(m, x[j]);
                if (x[j] > best) best = x[j], at = int32_t(i + j);
            }
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            m = __builtin_elementwise_maximum(m, __shfl_xor(m, o));
            take_larger(best, at, __shfl_xor(best, o), __shfl_xor(at, o));
        }
        if (lane == 0) sm[wave] = best, sa[wave] = at, ss[wave] = m == m ? 0.0 : __builtin_nan("");
        __syncthreads();
        if (threadIdx.x == 0) {
            double bad = ss[0];
            for (uint32_t w = 1; w < W; ++w) take_larger(best, at, sm[w], sa[w]), bad += ss[w];
            out[size_t(t) * sp.rows_n + blockIdx.x] = Slice{bad, best, at};
        }
        return;
    }
    // The sum over a reference: a logit of the first ones, raised where a later one is
    // 2^200 times as likely (2^1023 is fp64's end).
    constexpr uint32_t N = 8, STEP = N * kThreads;
    const float lead = float(200.0 / z.c);
    float ref = -3.4028235e38f, limit = ref;
    double sum = 0.0;
    auto add = [&](const float (&x)[N]) __attribute__((always_inline)) {
        float n = x[0];
#pragma unroll
        for (uint32_t j = 1; j < N; ++j) n = __builtin_elementwise_maximum(n, x[j]);
        m = __builtin_elementwise_maximum(m, n);
        if (n > limit) {
            sum *= share(ref, n, z);
            ref = n;
            limit = ref + lead;
        }
        double y[2] = {0.0, 0.0};
#pragma unroll
        for (uint32_t j = 0; j < N; ++j) y[j % 2] += power(__builtin_fmax(double(x[j]) - double(ref), z.least), z.c);
        sum += y[0] + y[1];
    };
    auto fetch = [&](uint32_t i, float (&x)[N]) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t h = 0; h < N / 4; ++h) {
            const f32x4u v = *reinterpret_cast<const f32x4u *>(l + i + 4 * (threadIdx.x + h * kThreads));
#pragma unroll
            for (int j = 0; j < 4; ++j) x[4 * h + j] = v[j];
        }
    };
    uint32_t i = i0;
    float next[N];
    if (i + STEP <= i1) fetch(i, next);
    for (; i + STEP <= i1; i += STEP) {
        float x[N];
#pragma unroll
        for (uint32_t j = 0; j < N; ++j) x[j] = next[j];
        // (the last again: what may not be under way could not be told from what is)
        fetch(i + 2 * STEP <= i1 ? i + STEP : i, next);
        __builtin_amdgcn_sched_barrier(0);
        add(x);
    }
    if (i < i1) {
        float x[N];
#pragma unroll
        for (uint32_t h = 0; h < N / 4; ++h) four(l, min(i + 4 * (threadIdx.x + h * kThreads), i1), i1, -kInf, x + 4 * h);
        add(x);
    }
    // the lanes' sums over the slice's largest
    float top = m;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = __builtin_elementwise_maximum(top, __shfl_xor(top, o));
    if (lane == 0) sm[wave] = top;
    __syncthreads();
    top = sm[0];
#pragma unroll
    for (uint32_t w = 1; w < W; ++w) top = __builtin_elementwise_maximum(top, sm[w]);
    sum = wave_sum(top > -kInf ? sum * share(ref, top, z) : 0.0);
    if (lane == 0) ss[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (uint32_t w = 1; w < W; ++w) sum += ss[w];
        // (a NaN's slice must not be the largest: -inf, and a sum that says so)
        out[size_t(t) * sp.rows_n + blockIdx.x] = top == top ? Slice{sum, top, 0} : Slice{__builtin_nan(""), -kInf, 0};
    }
}

// A whole row from its slices, by one wave; the same in every lane.
__device__ __forceinline__ Slice join(const Slice *r, uint32_t n, Scale z) {
    const uint32_t lane = threadIdx.x & 63;
    float m = -kInf;
    int32_t at = 0x7FFFFFFF;
    for (uint32_t i = lane; i < n; i += 64) take_larger(m, at, r[i].m, r[i].at);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) take_larger(m, at, __shfl_xor(m, o), __shfl_xor(at, o));
    double sum = 0.0;
    for (uint32_t i = lane; i < n; i += 64) sum += r[i].sum * (z.c != 0.0 && m > -kInf ? share(r[i].m, m, z) : 1.0);
    return Slice{wave_sum(sum), m, at};
}

// Sampling weight of token i with logit l at the stop: of the residual (over draft
// probability q, or without the draft itself), and of p alone. (Not contracted: a slice
// that has a weight in one kernel has it in the other.)
__device__ __forceinline__ Weight weight(const Stop &st, float l, float q, bool probs, uint32_t i, Scale z) {
#pragma clang fp contract(off)
    const double p = share(l, st.m, z) * st.inv;
    double r = p;
    if (probs)
        r = fmax(p - double(q), 0.0);
    else if (int32_t(i) == st.draft)
        r = 0.0;
    return Weight{r, p};
}

__global__ __launch_bounds__(kThreadsSeq, 6) void k_verify_weights(VerifyArgs a, Split sp, const Slice *__restrict__ rows,
                                                                Weight *__restrict__ out, Stop *__restrict__ stops) {
    constexpr uint32_t W = kThreadsSeq / 64;
    const uint32_t s = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __shared__ uint32_t first;
    __shared__ Stop stop;
    uint32_t b, e;
    seq_rows(a.start, a.n_tokens, s, &b, &e);
    const uint32_t n = e - b;
    const Scale z = scale_of(a.temperature[s]);
    if (n == 0) {
        if (threadIdx.x == 0 && blockIdx.x == 0) {
            a.n_accepted[s] = 0;
            a.next_token[s] = -1;
            stops[s] = Stop{0.0, 0.0f, -1, -1, 0};
        }
        return;
    }
    if (threadIdx.x == 0) first = n;
    __syncthreads();
    // a wave per row, up to its first that ends the chunk
    uint32_t i = wave;
    int32_t x = -1;
    bool good = false;
    Slice r{};
    for (; i < n; i += W) {
        bool inside = false;
        float lx = 0.0f, q = 1.0f, u = 0.0f;
        if (i + 1 < n) {
            x = a.tokens[b + i + 1];
            u = a.accept_u[b + i];
            inside = uint32_t(x) < a.vocab;
            const size_t at = size_t(b + i) * a.vocab + uint32_t(x);
            if (inside) lx = a.logits[at];
            if (inside && a.draft_probs != nullptr) q = a.draft_probs[at];
        }
        r = join(rows + size_t(b + i) * sp.rows_n, sp.rows_n, z);
        good = r.m > -kInf && r.m < kInf && r.sum == r.sum;
        bool take = good && inside;
        if (z.c == 0.0)
            take = take && x == r.at;
        else
            take = take && double(u) * double(q) < share(lx, r.m, z) / r.sum;
        if (!take) break;
    }
    if (i < n && lane == 0) atomicMin(&first, i);
    __syncthreads();
    if (i == first && lane == 0) {  // (one wave's, and every chunk ends with its last row at the latest)
        // (a draft outside the vocabulary equals no token)
        const int32_t draft = i + 1 < n ? int32_t(min(uint32_t(x), 0x7FFFFFFFu)) : -1;
        stop = Stop{1.0 / r.sum, r.m, int32_t(b + i), draft, good};
        if (blockIdx.x == 0) {
            stops[s] = stop;
            a.n_accepted[s] = int32_t(i);
            if (z.c == 0.0) a.next_token[s] = good ? r.at : -1;
        }
    }
    if (z.c == 0.0) return;
    __syncthreads();
    const Stop st = stop;
    const float *l = a.logits + size_t(st.row) * a.vocab;
    const float *q = a.draft_probs != nullptr && st.draft >= 0 ? a.draft_probs + size_t(st.row) * a.vocab : nullptr;
    // a wave per slice
    const uint32_t slice = blockIdx.x * W + wave;
    if (slice >= sp.pick_n) return;
    const uint32_t i0 = slice * sp.pick_len, i1 = min(i0 + sp.pick_len, a.vocab);
    double rest = 0.0, full = 0.0;
    for (uint32_t k = i0 + 4 * lane; k < i1; k += 256) {
        float y[4], d[4];
        four(l, k, i1, -kInf, y);
        if (q != nullptr) four(q, k, i1, 0.0f, d);
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            const Weight w = weight(st, y[j], q != nullptr ? d[j] : 0.0f, q != nullptr, k + j, z);
            rest += w.rest;
            full += w.full;
        }
    }
    rest = wave_sum(rest);
    full = wave_sum(full);
    if (lane == 0) out[size_t(s) * sp.pick_n + slice] = Weight{rest, full};
}

// Twice the same: the first entry whose running sum passes a goal, the last one of any
// weight where none does (a random number next to 1, and roundings); over the row's
// slices, by each wave for itself, then over the slice's tokens. A thread's entries lie
// next to each other. Where a lane's sums begin may differ by roundings from where the
// last lane's ended, so that a goal between the two is passed before the first slice of
// the next lane: its first weight is the one then, as for random numbers below 0.
__global__ __launch_bounds__(kThreadsPick) void k_verify_pick(VerifyArgs a, Split sp, const Weight *__restrict__ w,
                                                             const Stop *__restrict__ stops) {
    constexpr uint32_t W = kThreadsPick / 64;
    const uint32_t s = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    __shared__ double waves[W];
    __shared__ uint32_t ends[W];
    const Weight *r = w + size_t(s) * sp.pick_n;
    const uint32_t slices = div_up(sp.pick_n, 64);
    const uint32_t b0 = min(lane * slices, sp.pick_n), e0 = min(b0 + slices, sp.pick_n);
    const double u = a.sample_u[s];
    const Scale z = scale_of(a.temperature[s]);
    const Stop st = stops[s];
    double rest = 0.0, full = 0.0;  // (of anything where there is nothing to pick; unused then)
#pragma unroll 4
    for (uint32_t i = b0; i < e0; ++i) rest += r[i].rest, full += r[i].full;
    if (st.row < 0 || z.c == 0.0) return;
    if (!st.good) {
        if (tid == 0) a.next_token[s] = -1;
        return;
    }
    const double rest_to = wave_scan(rest), full_to = wave_scan(full), all_rest = lane_value(rest_to, 63);
    const bool residual = all_rest > 0.0;
    double goal = u * (residual ? all_rest : lane_value(full_to, 63));
    double before = residual ? rest_to - rest : full_to - full, at = 0.0;
    uint32_t hit = 0xFFFFFFFFu, mine = 0;
#pragma unroll 4
    for (uint32_t i = b0; i < e0; ++i) {
        const double v = residual ? r[i].rest : r[i].full;
        if (v > 0.0) {
            if (hit == 0xFFFFFFFFu && before + v > goal) hit = i, at = before;
            mine = i + 1;
        }
        before += v;
    }
    const uint64_t hits = __ballot(hit != 0xFFFFFFFFu), any = __ballot(mine != 0);
    if (any == 0) {  // (cannot be: the row's weights sum to 1)
        if (tid == 0) a.next_token[s] = -1;
        return;
    }
    const uint32_t from = hits != 0 ? __builtin_ctzll(hits) : 63 - __builtin_clzll(any);
    const uint32_t slice = hits != 0 ? __builtin_amdgcn_readlane(hit, from) : __builtin_amdgcn_readlane(mine, from) - 1;
    // (not below 0, which no weight would be the first to pass; no token of the last slice
    // passes infinity)
    goal = hits != 0 ? __builtin_fmax(goal - lane_value(at, from), 0.0) : __builtin_inf();

    const float *l = a.logits + size_t(st.row) * a.vocab;
    const float *q = a.draft_probs != nullptr && st.draft >= 0 ? a.draft_probs + size_t(st.row) * a.vocab : nullptr;
    // a wave's tokens lie next to each other, 256 of them at a time
    const uint32_t end = min(slice * sp.pick_len + sp.pick_len, a.vocab), per = div_up(sp.pick_len, 4 * W) * 4;
    const uint32_t i0 = min(slice * sp.pick_len + wave * per, end), i1 = min(i0 + per, end);
    auto values = [&](uint32_t i, double *v) __attribute__((always_inline)) {
        float y[4], d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        four(l, i, i1, -kInf, y);
        if (q != nullptr) four(q, i, i1, 0.0f, d);
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            const Weight x = weight(st, y[j], d[j], q != nullptr, i + j, z);
            v[j] = residual ? x.rest : x.full;
        }
    };
    double sum = 0.0;
    mine = 0;
#pragma unroll 2
    for (uint32_t i = i0 + 4 * lane; i < i1; i += 256) {
        double v[4];
        values(i, v);
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            if (v[j] > 0.0) mine = i + j + 1;
            sum += v[j];
        }
    }
    sum = wave_sum(sum);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mine = max(mine, uint32_t(__shfl_xor(int(mine), o)));
    if (lane == 0) waves[wave] = sum, ends[wave] = mine;
    __syncthreads();
    before = 0.0;
    for (uint32_t k = 0; k < wave; ++k) before += waves[k];
    const bool here = mine != 0 && !(before > goal) && before + sum > goal;  // (one wave's at most)
    bool later = false;  // whether some wave passes the goal
    double run = 0.0;
    for (uint32_t k = 0; k < W; ++k) run += waves[k], later = later || (ends[k] != 0 && run > goal);
    if (here) {
        uint32_t token = mine - 1;
        for (uint32_t i = i0; i < i1; i += 256) {
            double v[4];
            values(min(i + 4 * lane, i1), v);
            const double upto = wave_scan(v[0] + v[1] + v[2] + v[3]);
            double x = before + lane_value(upto, 63);
            if (x > goal) {
                x = before + (upto - (v[0] + v[1] + v[2] + v[3]));
                uint32_t first = 4;
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) {
                    x += v[j];
                    if (first == 4 && v[j] > 0.0 && x > goal) first = j;
                }
                const uint64_t hits = __ballot(first < 4);
                if (hits != 0) {
                    const uint32_t from = __builtin_ctzll(hits);
                    token = i + 4 * from + __builtin_amdgcn_readlane(first, from);
                    break;
                }
            }
            before += lane_value(upto, 63);
        }
        if (lane == 0) a.next_token[s] = int32_t(token);
    } else if (!later && tid == 0) {
        uint32_t last = 1;
        for (uint32_t k = 0; k < W; ++k) last = max(last, ends[k]);
        a.next_token[s] = int32_t(last - 1);
    }
}

size_t up(size_t v) { return (v + 255) & ~size_t(255); }

}  // namespace

// For any vocabulary: a slice of each row, or as many as make kRowsPerCu (kPickPerCu) per CU.
size_t verify_scratch_bytes(uint32_t n_tokens, uint32_t n_seq) {
    return up(std::max(kRowsPerCu * kMostCu, n_tokens) * sizeof(Slice)) + up(std::max(kPickPerCu * kMostCu, n_seq) * sizeof(Weight)) +
           up(n_seq * sizeof(Stop));
}

hipError_t launch_verify(const VerifyArgs &a, int num_cu, void *scratch, hipStream_t st) {
    const Split sp = split(a.vocab, a.n_tokens, a.n_seq, std::min(num_cu, kMostCu));
    char *p = static_cast<char *>(scratch);
    Slice *rows = reinterpret_cast<Slice *>(p);
    p += up(std::max(kRowsPerCu * kMostCu, a.n_tokens) * sizeof(Slice));
    Weight *w = reinterpret_cast<Weight *>(p);
    p += up(std::max(kPickPerCu * kMostCu, a.n_seq) * sizeof(Weight));
    Stop *stops = reinterpret_cast<Stop *>(p);
    k_verify_rows<<<dim3(sp.rows_n, a.n_tokens), kThreads, 0, st>>>(a, sp, rows);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    k_verify_weights<<<dim3(div_up(sp.pick_n, kThreadsSeq / 64), a.n_seq), kThreadsSeq, 0, st>>>(a, sp, rows, w, stops);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    k_verify_pick<<<a.n_seq, kThreadsPick, 0, st>>>(a, sp, w, stops);
    return hipGetLastError();
}

}  // namespace tc
