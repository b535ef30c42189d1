// tc_verify.hip -- verification of drafted tokens against the target's logits.
//
// Three launches. k_verify_rows reads every logit once: for a slice of a row the
// largest and, over it, the sum of exponentials (where the temperature is 0: the
// largest's lowest index). k_verify_weights joins a sequence's slices, walks its
// drafts, and sums the sampling weights of the row where they end, again in slices;
// k_verify_pick finds the slice and then the token that the random number falls on.
// The first is bound by HBM and by fp64 arithmetic about alike, the others by
// their latency.
//
// Everything behind the logits is fp64: a token's probability in a vocabulary of
// 10^5 is 10^-5 and less, so sums in fp32 would move the borders between tokens by
// a hundredth of their width.
#include "tc_attn_common.hpp"
#include "tc_kernels.hpp"

namespace tc {
namespace {

constexpr uint32_t kThreads = 256, kWaves = kThreads / 64;

// (4-byte aligned: rows of an odd vocabulary)
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

// A slice of a row: its largest logit, that logit's lowest index, and the sum of
// exp((l - m) / temperature). NaN logits give a NaN sum.
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

// Slices of at least 1024 logits (4 loads of a thread), as many as give each CU
// four workgroups.
Split split(uint32_t vocab, uint32_t n_tokens, uint32_t n_seq, int num_cu) {
    const uint32_t want = 4 * uint32_t(num_cu), most = div_up(vocab, 1024);
    auto slices = [&](uint32_t rows) {
        const uint32_t n = div_up(want, rows);
        return n < most ? n : most;
    };
    Split s;
    s.rows_len = div_up(div_up(vocab, slices(n_tokens)), 4) * 4;
    s.rows_n = div_up(vocab, s.rows_len);
    s.pick_len = div_up(div_up(vocab, slices(n_seq)), 4) * 4;
    s.pick_n = div_up(vocab, s.pick_len);
    return s;
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// 1 / temperature, 0 for the greedy choice.
__device__ __forceinline__ double inverse_temperature(float t) { return t > 0.0f ? 1.0 / double(t) : 0.0; }

// (m, at) of the larger logit, the lower index where they are alike.
__device__ __forceinline__ void take_larger(float &m, int32_t &at, float om, int32_t oat) {
    if (om > m || (om == m && oat < at)) m = om, at = oat;
}

__global__ __launch_bounds__(kThreads) void k_verify_rows(VerifyArgs a, Split sp, Slice *__restrict__ out) {
    const uint32_t t = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int s = find_seq(a.start, a.n_seq, t);
    if (s < 0) return;
    const double it = inverse_temperature(a.temperature[s]);
    const float *l = a.logits + size_t(t) * a.vocab;
    const uint32_t i0 = blockIdx.x * sp.rows_len, i1 = min(i0 + sp.rows_len, a.vocab);
    float m = -__builtin_inff();
    int32_t at = 0x7FFFFFFF;
    double sum = 0.0;
    for (uint32_t i = i0 + 4 * threadIdx.x; i < i1; i += 4 * kThreads) {
        float x[4];
        if (i + 4 <= i1) {
            const f32x4u v = *reinterpret_cast<const f32x4u *>(l + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = v[j];
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = i + j < i1 ? l[i + j] : -__builtin_inff();
        }
        float n = m;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (x[j] > n) n = x[j], at = int32_t(i + j);
        if (n > m) {  // (from -inf: the sum is 0 and stays so)
            sum = m > -__builtin_inff() ? sum * exp((double(m) - double(n)) * it) : sum;
            m = n;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (!(x[j] == -__builtin_inff())) sum += exp((double(x[j]) - double(m)) * it);
    }
    // the lanes' sums over the slice's largest
    __shared__ float sm[kWaves];
    __shared__ int32_t sa[kWaves];
    __shared__ double ss[kWaves];
    float wm = m;
    int32_t wat = at;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) take_larger(wm, wat, __shfl_xor(wm, o), __shfl_xor(wat, o));
    if (lane == 0) sm[wave] = wm, sa[wave] = wat;
    __syncthreads();
    wm = sm[0], wat = sa[0];
    for (uint32_t w = 1; w < kWaves; ++w) take_larger(wm, wat, sm[w], sa[w]);
    if (m > -__builtin_inff()) sum *= exp((double(m) - double(wm)) * it);
    sum = wave_sum(sum);
    if (lane == 0) ss[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        double r = ss[0];
        for (uint32_t w = 1; w < kWaves; ++w) r += ss[w];
        out[size_t(t) * sp.rows_n + blockIdx.x] = Slice{r, wm, wat};
    }
}

// A whole row from its slices, by one wave; the same in every lane.
__device__ __forceinline__ Slice join(const Slice *r, uint32_t n, double it) {
    const uint32_t lane = threadIdx.x & 63;
    float m = -__builtin_inff();
    int32_t at = 0x7FFFFFFF;
    for (uint32_t i = lane; i < n; i += 64) take_larger(m, at, r[i].m, r[i].at);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) take_larger(m, at, __shfl_xor(m, o), __shfl_xor(at, o));
    double sum = 0.0;
    for (uint32_t i = lane; i < n; i += 64) {
        const Slice q = r[i];
        if (q.m > -__builtin_inff())
            sum += q.sum * exp((double(q.m) - double(m)) * it);
        else
            sum += q.sum;  // 0, or a NaN
    }
    return Slice{wave_sum(sum), m, at};
}

// Sampling weight of token i at the stop: of the residual, and of p alone.
__device__ __forceinline__ Weight weight(const Stop &st, const float *l, const float *q, uint32_t i, double it) {
    const double p = exp((double(l[i]) - double(st.m)) * it) * st.inv;
    double r = p;
    if (st.draft >= 0) {
        if (q != nullptr)
            r = fmax(p - double(q[i]), 0.0);
        else if (int32_t(i) == st.draft)
            r = 0.0;
    }
    return Weight{r, p};
}

__global__ __launch_bounds__(kThreads) void k_verify_weights(VerifyArgs a, Split sp, const Slice *__restrict__ rows,
                                                             Weight *__restrict__ out, Stop *__restrict__ stops) {
    const uint32_t s = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __shared__ uint32_t first;
    __shared__ Stop stop;
    __shared__ double sr[kWaves], sf[kWaves];
    uint32_t b, e;
    seq_rows(a.start, a.n_tokens, s, &b, &e);
    const uint32_t n = e - b;
    const float temp = a.temperature[s];
    const double it = inverse_temperature(temp);
    if (threadIdx.x == 0) {
        first = n;
        stop = Stop{0.0, 0.0f, -1, -1, 0};
    }
    __syncthreads();
    // a wave per row; the first row that ends the chunk
    for (uint32_t i = wave; i < n; i += kWaves) {
        const Slice r = join(rows + size_t(b + i) * sp.rows_n, sp.rows_n, it);
        const bool good = r.m > -__builtin_inff() && r.m < __builtin_inff() && r.sum == r.sum;
        bool end = i + 1 == n;
        const int32_t x = end ? -1 : a.tokens[b + i + 1];
        if (!end) {
            bool take = false;
            if (good && uint32_t(x) < a.vocab) {
                if (it == 0.0) {
                    take = x == r.at;
                } else {
                    const size_t at = size_t(b + i) * a.vocab + uint32_t(x);
                    const double p = exp((double(a.logits[at]) - double(r.m)) * it) / r.sum;
                    const double q = a.draft_probs != nullptr ? double(a.draft_probs[at]) : 1.0;
                    take = double(a.accept_u[b + i]) * q < p;
                }
            }
            end = !take;
        }
        if (end && lane == 0) atomicMin(&first, i);
    }
    __syncthreads();
    if (n != 0 && wave == 0) {
        const uint32_t i = first;
        const Slice r = join(rows + size_t(b + i) * sp.rows_n, sp.rows_n, it);
        if (lane == 0) {
            stop.good = r.m > -__builtin_inff() && r.m < __builtin_inff() && r.sum == r.sum;
            stop.inv = 1.0 / r.sum;
            stop.m = r.m;
            stop.row = int32_t(b + i);
            if (i + 1 < n) {  // (a draft outside the vocabulary equals no token)
                const uint32_t x = uint32_t(a.tokens[b + i + 1]);
                stop.draft = int32_t(min(x, 0x7FFFFFFFu));
            }
            if (blockIdx.x == 0) {
                a.n_accepted[s] = int32_t(i);
                if (it == 0.0) a.next_token[s] = stop.good ? r.at : -1;
            }
        }
    } else if (n == 0 && threadIdx.x == 0 && blockIdx.x == 0) {
        a.n_accepted[s] = 0;
        a.next_token[s] = -1;
    }
    __syncthreads();
    const Stop st = stop;
    if (blockIdx.x == 0 && threadIdx.x == 0) stops[s] = st;
    if (st.row < 0 || it == 0.0) return;
    const float *l = a.logits + size_t(st.row) * a.vocab;
    const float *q = a.draft_probs != nullptr ? a.draft_probs + size_t(st.row) * a.vocab : nullptr;
    const uint32_t i0 = blockIdx.x * sp.pick_len, i1 = min(i0 + sp.pick_len, a.vocab);
    double rest = 0.0, full = 0.0;
    for (uint32_t i = i0 + threadIdx.x; i < i1; i += kThreads) {
        const Weight w = weight(st, l, q, i, it);
        rest += w.rest;
        full += w.full;
    }
    rest = wave_sum(rest);
    full = wave_sum(full);
    if (lane == 0) sr[wave] = rest, sf[wave] = full;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (uint32_t w = 1; w < kWaves; ++w) rest += sr[w], full += sf[w];
        out[size_t(s) * sp.pick_n + blockIdx.x] = Weight{rest, full};
    }
}

__global__ __launch_bounds__(kThreads) void k_verify_pick(VerifyArgs a, Split sp, const Weight *__restrict__ w,
                                                          const Stop *__restrict__ stops) {
    const uint32_t s = blockIdx.x, tid = threadIdx.x;
    const Stop st = stops[s];
    const double it = inverse_temperature(a.temperature[s]);
    if (st.row < 0 || it == 0.0) return;
    if (!st.good) {
        if (tid == 0) a.next_token[s] = -1;
        return;
    }
    __shared__ uint32_t slice;
    __shared__ double target;
    __shared__ int residual;
    __shared__ double sums[kThreads];
    __shared__ uint32_t found, last;
    const Weight *r = w + size_t(s) * sp.pick_n;
    if (tid == 0) {
        double rest = 0.0, full = 0.0;
        for (uint32_t i = 0; i < sp.pick_n; ++i) rest += r[i].rest, full += r[i].full;
        residual = rest > 0.0;
        const double all = residual ? rest : full;
        const double goal = double(a.sample_u[s]) * all;
        // the slice where the running sum passes the goal; the last of any
        // weight where none does
        double before = 0.0, base = 0.0;
        uint32_t at = 0;
        bool hit = false;
        for (uint32_t i = 0; i < sp.pick_n && !hit; ++i) {
            const double x = residual ? r[i].rest : r[i].full;
            if (x > 0.0) at = i, base = before;
            hit = before + x > goal;
            before += x;
        }
        slice = at;
        target = goal - base;
        found = 0xFFFFFFFFu;
        last = 0;
    }
    __syncthreads();
    const float *l = a.logits + size_t(st.row) * a.vocab;
    const float *q = a.draft_probs != nullptr ? a.draft_probs + size_t(st.row) * a.vocab : nullptr;
    const uint32_t i0 = slice * sp.pick_len, i1 = min(i0 + sp.pick_len, a.vocab);
    const uint32_t per = div_up(sp.pick_len, kThreads);
    const uint32_t b = min(i0 + tid * per, i1), e = min(b + per, i1);
    double sum = 0.0;
    uint32_t mine = 0;
    for (uint32_t i = b; i < e; ++i) {
        const Weight x = weight(st, l, q, i, it);
        const double v = residual ? x.rest : x.full;
        if (v > 0.0) mine = i + 1;
        sum += v;
    }
    sums[tid] = sum;
    if (mine != 0) atomicMax(&last, mine);
    __syncthreads();
    double before = 0.0;
    for (uint32_t i = 0; i < tid; ++i) before += sums[i];
    if (before <= target && before + sum > target) {
        for (uint32_t i = b; i < e; ++i) {
            const Weight x = weight(st, l, q, i, it);
            const double v = residual ? x.rest : x.full;
            before += v;
            if (v > 0.0 && before > target) {
                atomicMin(&found, i);
                break;
            }
        }
    }
    __syncthreads();
    if (tid == 0) a.next_token[s] = int32_t(found != 0xFFFFFFFFu ? found : last - 1);
}

size_t up(size_t v) { return (v + 255) & ~size_t(255); }

}  // namespace

// For any vocabulary: the slices of both kernels are fewest rows' or four per CU.
size_t verify_scratch_bytes(uint32_t n_tokens, uint32_t n_seq) {
    constexpr size_t kMostCu = 256;
    return up((4 * kMostCu + n_tokens) * sizeof(Slice)) + up((4 * kMostCu + n_seq) * sizeof(Weight)) + up(n_seq * sizeof(Stop));
}

hipError_t launch_verify(const VerifyArgs &a, int num_cu, void *scratch, hipStream_t st) {
    const Split sp = split(a.vocab, a.n_tokens, a.n_seq, num_cu < 256 ? num_cu : 256);
    char *p = static_cast<char *>(scratch);
    Slice *rows = reinterpret_cast<Slice *>(p);
    p += up((1024 + a.n_tokens) * sizeof(Slice));
    Weight *w = reinterpret_cast<Weight *>(p);
    p += up((1024 + size_t(a.n_seq)) * sizeof(Weight));
    Stop *stops = reinterpret_cast<Stop *>(p);
    k_verify_rows<<<dim3(sp.rows_n, a.n_tokens), kThreads, 0, st>>>(a, sp, rows);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    k_verify_weights<<<dim3(sp.pick_n, a.n_seq), kThreads, 0, st>>>(a, sp, rows, w, stops);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    k_verify_pick<<<a.n_seq, kThreads, 0, st>>>(a, sp, w, stops);
    return hipGetLastError();
}

}  // namespace tc
