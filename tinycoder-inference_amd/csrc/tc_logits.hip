// tc_logits.hip -- penalties for repeated tokens, biases and masks on logits.
//
// A workgroup has a chunk of the vocabulary for one sequence. It counts the sequence's history
// there in LDS (integer sums, so their order changes nothing), adds up the biases in their
// order, and then takes the sequence's rows one after the other, each row's own token counted
// on top (as seen alone while it is the prompt's): every logit is read and written once, with its count and bias out of LDS beside it.
// Bound by HBM for many rows (219 of 152064 logits with masks: 57 to 58 us, 272 MB at 4.7
// TB/s; VALU 0.30 busy); for few by the chain lists' borders -> history -> LDS -> stores (one row 4.1
// us), and between these by the history, which every chunk's workgroup reads (256 rows of 32003
// 18 us, 15 without it, 10 for the bytes).
//
// No list of tokens is sorted and no counts are kept in HBM: a table of counts of one sequence
// would be as large as a row of its logits. More tokens of a lane were slower (219 rows 72 us
// with 16, 65 with 8), fewer lanes too (66 with 256 to a workgroup, which then counts more histories; one
// row 4.7 for 4.3), stores past the caches too once their reader was counted (131 -> 136 us with
// tc_spec_verify behind, 200 rows).
#include "tc_kernels.hpp"
#include "tc_step.hpp"

namespace tc {
namespace {

constexpr uint32_t kThreads = 512, kWaves = kThreads / 64;
constexpr uint32_t kSeen = 0x80000000u;  // in a count: the token is in the history
constexpr float kInf = __builtin_inff();

// (aligned to their elements: rows of an odd vocabulary, histories from any token on)
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t u16x4u __attribute__((ext_vector_type(4), aligned(2)));

__device__ __forceinline__ float widened(int type, uint32_t w) {
    return type == kF16 ? h2f(w) : __builtin_bit_cast(float, w << 16);
}

// Part [begin, end) of entry s in a list of n, kept inside it whatever `start` holds.
__device__ __forceinline__ void part_of(const int32_t *start, uint32_t s, uint32_t n, uint32_t *begin, uint32_t *end) {
    const int32_t N = int32_t(n), x = start[s], y = start[s + 1];
    const int32_t b = x < 0 ? 0 : x > N ? N : x;
    const int32_t e = y < b ? b : y > N ? N : y;
    *begin = uint32_t(b);
    *end = uint32_t(e);
}

// A sequence's penalties. The logit is divided by the repetition's factor as a product with its
// reciprocal in fp64, a step or two of fp64 from the quotient: where any lane of a wave has a
// token that was seen, all of them wait for it, and a division takes as long as the rest.
struct Penalties {
    double rep, inv_rep, freq, pres;
};
// A token's logit where rules change it.
__device__ __forceinline__ float changed(float l, uint32_t count, float bias, const Penalties &p) {
    double v = l;
    if (count != 0) {
        const uint32_t c = count & ~kSeen;
        v *= v > 0.0 ? p.inv_rep : p.rep;
        if (c != 0) v -= __builtin_fma(p.freq, double(c), p.pres);
    }
    return float(v + double(bias));
}

// 4 logits from token `i` of the chunk on (n: the chunk's), zeros behind its end.
template <int XT>
__device__ __forceinline__ void load4(const void *logits, uint64_t from, uint32_t i, uint32_t n, float (&l)[4]) {
    const bool whole = i + 4 <= n;
    if constexpr (XT == kF32) {
        const float *p = static_cast<const float *>(logits) + from + i;
        if (whole) {
            const f32x4u v = *reinterpret_cast<const f32x4u *>(p);
#pragma unroll
            for (int j = 0; j < 4; ++j) l[j] = v[j];
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) l[j] = i + j < n ? p[j] : 0.0f;
        }
    } else {
        const uint16_t *p = static_cast<const uint16_t *>(logits) + from + i;
        if (whole) {
            const u16x4u v = *reinterpret_cast<const u16x4u *>(p);
#pragma unroll
            for (int j = 0; j < 4; ++j) l[j] = widened(XT, v[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) l[j] = i + j < n ? widened(XT, p[j]) : 0.0f;
        }
    }
}

// The words of a row's mask from token lo on, null: no mask.
__device__ __forceinline__ const uint32_t *mask_of_row(const tc_logit_rules &r, uint32_t row, uint32_t lo) {
    if (!r.mask) return nullptr;
    const uint32_t m = r.mask_of ? uint32_t(r.mask_of[row]) : row;
    return m < r.n_masks ? r.mask + size_t(m) * r.mask_words + (lo >> 5) : nullptr;
}

// V: vectors of 4 logits that a lane has of its chunk.
template <int XT, int V>
__global__ __launch_bounds__(kThreads) void k_logits(LogitCall a) {
    constexpr uint32_t chunk = kThreads * 4 * V, step = kThreads * 4;
    extern __shared__ uint32_t lds[];
    uint32_t *counts = lds;
    float *bias = reinterpret_cast<float *>(lds + chunk);
    const uint32_t s = blockIdx.y, lo = blockIdx.x * chunk, n = min(chunk, a.vocab - lo);
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // everything that other loads wait for, side by side
    uint32_t begin, end, h0 = 0, h1 = 0, b0 = 0, b1 = 0;
    seq_rows(a.start, a.n_tokens, s, &begin, &end);
    uint32_t row = begin + blockIdx.z;
    const float rep = a.r.repetition ? a.r.repetition[s] : 1.0f, freq = a.r.frequency ? a.r.frequency[s] : 0.0f;
    const float pres = a.r.presence ? a.r.presence[s] : 0.0f;
    if (a.r.history_start) part_of(a.r.history_start, s, a.r.n_history, &h0, &h1);
    if (a.r.bias_start) part_of(a.r.bias_start, s, a.r.n_bias, &b0, &b1);
    const int32_t asked = a.r.prompt ? a.r.prompt[s] : 0;
    if (row >= end) return;
    const bool counted = rep != 1.0f || freq != 0.0f || pres != 0.0f, biased = b0 != b1;
    if (!counted) h1 = h0;
    // tokens that were asked: of the history those before `answers`, and of the rows' own, where
    // the number goes on over them (below 0), the first asked_rows
    const uint32_t ask = asked < 0 ? 0u - uint32_t(asked) : uint32_t(asked), past = min(ask, h1 - h0);
    const uint32_t answers = h0 + past, asked_rows = asked < 0 ? ask - past : 0;
    // the first row is on its way while the history is counted, each other one while the row
    // before it is worked on
    float l[V][4];
    uint32_t words[V];
    auto load = [&](uint32_t r) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const uint32_t i = tid * 4 + v * step;
            if (i < n) load4<XT>(a.logits, r * a.x_stride + lo, i, n, l[v]);
        }
        const uint32_t *mask = mask_of_row(a.r, r, lo);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const uint32_t i = tid * 4 + v * step;
            words[v] = ~0u;
            if (mask && i < n) words[v] = mask[i >> 5];
        }
    };
    // each lane's first four tokens of the history and its first of the biases; at the end of all
    // histories the last four, of which a lane counts its own (219 rows 64.7 -> 64.4 us, one row 4.3 ->
    // 4.1 with 16 bytes a load instead of 4)
    auto four = [&](uint32_t i) { return u32x4(*reinterpret_cast<const u32x4u *>(a.r.history + min(i, a.r.n_history - 4))); };
    u32x4 first = {0, 0, 0, 0};
    if (h0 != h1 && a.r.n_history >= 4) first = four(h0 + 4 * tid);
    uint32_t bias_token = b0 + lane < b1 ? uint32_t(a.r.bias_token[b0 + lane]) : ~0u;
    float bias_value = b0 + lane < b1 ? a.r.bias_value[b0 + lane] : 0.0f;
    load(row);
    const u32x4 zero = {0, 0, 0, 0};
    if (counted)
#pragma unroll
        for (int v = 0; v < V; ++v) *reinterpret_cast<u32x4 *>(counts + tid * 4 + v * step) = zero;
    if (biased)
#pragma unroll
        for (int v = 0; v < V; ++v) *reinterpret_cast<u32x4 *>(lds + chunk + tid * 4 + v * step) = zero;
    __syncthreads();
    auto count = [&](int32_t token, bool only_seen) {
        const uint32_t t = uint32_t(token) - lo;
        if (t < n) {
            if (only_seen)
                atomicOr(counts + t, kSeen);
            else
                atomicAdd(counts + t, 1u);
        }
    };
    auto count4 = [&](const u32x4 &t, uint32_t i) {
        const uint32_t at = min(i, a.r.n_history - 4);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (at + j >= i && at + j < h1) count(int32_t(t[j]), at + j < answers);
    };
    uint32_t i = h0 + 4 * tid;
    if (a.r.n_history >= 4) {
        if (h0 != h1) {
            count4(first, i);
            for (i += 4 * kThreads; i < h1; i += 8 * kThreads) {
                u32x4 t[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) t[j] = four(i + j * 4 * kThreads);
#pragma unroll
                for (int j = 0; j < 2; ++j) count4(t[j], i + j * 4 * kThreads);
            }
        }
    } else {
        for (i = h0 + tid; i < h1; i += kThreads) count(a.r.history[i], i < answers);
    }
    if (biased) {
        // each wave has a part of the chunk, and adds the biases there one after the other
        constexpr uint32_t part = chunk / kWaves;
        const uint32_t p0 = lo + wave * part;
        for (uint32_t i0 = b0;;) {
            const uint32_t t = bias_token - p0;
            for (uint64_t m = __ballot(t < part && bias_token < a.vocab); m != 0; m &= m - 1) {
                const int b = __builtin_ctzll(m);
                const uint32_t at = wave * part + __builtin_amdgcn_readlane(t, b);
                const float add = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, bias_value), b));
                if (lane == 0) bias[at] += add;
            }
            if ((i0 += 64) >= b1) break;
            const uint32_t i = i0 + lane;
            bias_token = i < b1 ? uint32_t(a.r.bias_token[i]) : ~0u;
            bias_value = i < b1 ? a.r.bias_value[i] : 0.0f;
        }
    }
    __syncthreads();
    const Penalties p{double(rep), 1.0 / double(rep), double(freq), double(pres)};
    const bool own_tokens = counted && a.tokens;
    for (uint32_t told = begin; row < end; row += gridDim.z) {
        if (own_tokens) {
            for (told += tid; told <= row; told += kThreads) count(a.tokens[told], told - begin < asked_rows);
            told = row + 1;
            __syncthreads();
        }
        float *out = a.out + row * a.out_stride + lo;
        float o[V][4];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const uint32_t i = tid * 4 + v * step, allowed = words[v] >> (i & 31);
            u32x4 c = zero;
            f32x4 b = {0.0f, 0.0f, 0.0f, 0.0f};
            if (counted) c = *reinterpret_cast<const u32x4 *>(counts + i);
            if (biased) b = *reinterpret_cast<const f32x4 *>(bias + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                o[v][j] = l[v][j];
                if (c[j] != 0 || b[j] != 0.0f) o[v][j] = changed(l[v][j], c[j], b[j], p);
                if (!(allowed >> j & 1)) o[v][j] = -kInf;
            }
        }
        if (row + gridDim.z < end) load(row + gridDim.z);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const uint32_t i = tid * 4 + v * step;
            if (i + 4 <= n) {
                *reinterpret_cast<f32x4u *>(out + i) = f32x4u{o[v][0], o[v][1], o[v][2], o[v][3]};
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (i + j < n) out[i + j] = o[v][j];
            }
        }
        if (own_tokens) __syncthreads();
    }
}

template <int XT, int V>
hipError_t launch(const LogitCall &c, uint32_t parts, hipStream_t st) {
    const uint32_t chunk = kThreads * 4 * V, bytes = chunk * (c.r.bias_start ? 8 : 4);
    k_logits<XT, V><<<dim3((c.vocab + chunk - 1) / chunk, c.n_seq, parts), kThreads, bytes, st>>>(c);
    return hipGetLastError();
}
template <int XT>
hipError_t launch(const LogitCall &c, int num_cu, hipStream_t st) {
    // Chunks of 4096 tokens where those of 2048 are more than 2 to a CU (6 rows of each of 8 sequences of
    // 152064: 13.7 us, 16.1 with 2048; 4 sequences of a row 5.1 and 4.95); a sequence's rows by several
    // workgroups, each of which counts the history, up to 4 to a CU (6 rows of each of 4 sequences
    // 10.3 us, 12.9 with up to 2, 11.8 with up to 8).
    const uint64_t cu = num_cu, chunks = uint64_t((c.vocab + 2047) / 2048) * c.n_seq;
    const bool wide = chunks > 2 * cu;
    const uint64_t most = (c.n_tokens + c.n_seq - 1) / c.n_seq, fill = 4 * cu / (wide ? (chunks + 1) / 2 : chunks);
    const uint32_t parts = uint32_t(fill < 1 ? 1 : fill < most ? fill : most);
    return wide ? launch<XT, 2>(c, parts, st) : launch<XT, 1>(c, parts, st);
}

}  // namespace

hipError_t launch_logits(const LogitCall &c, int num_cu, hipStream_t st) {
    switch (c.xtype) {
        case kF32: return launch<kF32>(c, num_cu, st);
        case kF16: return launch<kF16>(c, num_cu, st);
        default: return launch<kBF16>(c, num_cu, st);
    }
}

}  // namespace tc
