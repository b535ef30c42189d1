// tc_logits.hip -- penalties for repeated tokens, biases and masks on logits.
//
// A workgroup has a chunk of the vocabulary for one sequence. It counts the sequence's history
// there in LDS (integer sums, so their order changes nothing), adds up the biases in their
// order, and then takes the sequence's rows one after the other, each row's own token counted
// on top: every logit is read and written once, with its count and bias out of LDS beside it.
// Bound by HBM for many rows; for few by the history, which each chunk's workgroup reads.
//
// No list of tokens is sorted and no counts are kept in HBM: a table of counts of one sequence
// would be as large as a row of its logits.
#include <algorithm>

#include "tc_kernels.hpp"
#include "tc_step.hpp"

namespace tc {
namespace {

constexpr uint32_t kThreads = 256, kWaves = kThreads / 64;
constexpr uint32_t kSeen = 0x80000000u;  // in a count: the token is in the history
constexpr float kInf = __builtin_inff();

// (aligned to their elements: rows of an odd vocabulary)
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
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

// A token's logit where rules change it.
__device__ __forceinline__ float changed(float l, uint32_t count, float bias, float rep, float freq, float pres) {
    double v = l;
    if (count != 0) {
        const uint32_t c = count & ~kSeen;
        v = v > 0.0 ? v / double(rep) : v * double(rep);
        if (c != 0) v -= double(freq) * double(c) + double(pres);
    }
    return float(v + double(bias));
}

__global__ __launch_bounds__(kThreads) void k_logits(LogitCall a) {
    extern __shared__ uint32_t lds[];
    uint32_t *counts = lds;
    float *bias = reinterpret_cast<float *>(lds + a.chunk);
    const uint32_t s = blockIdx.y, lo = blockIdx.x * a.chunk, n = min(a.chunk, a.vocab - lo);
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint32_t row, end;
    seq_rows(a.start, a.n_tokens, s, &row, &end);
    if (row == end) return;
    const float rep = a.r.repetition ? a.r.repetition[s] : 1.0f, freq = a.r.frequency ? a.r.frequency[s] : 0.0f;
    const float pres = a.r.presence ? a.r.presence[s] : 0.0f;
    const bool counted = rep != 1.0f || freq != 0.0f || pres != 0.0f;
    uint32_t b0 = 0, b1 = 0;
    if (a.r.bias_start) part_of(a.r.bias_start, s, a.r.n_bias, &b0, &b1);
    const bool biased = b0 != b1;
    if (counted)
        for (uint32_t i = tid; i < a.chunk; i += kThreads) counts[i] = 0;
    if (biased)
        for (uint32_t i = tid; i < a.chunk; i += kThreads) bias[i] = 0.0f;
    __syncthreads();
    if (counted && a.r.history_start) {
        uint32_t h0, h1;
        part_of(a.r.history_start, s, a.r.n_history, &h0, &h1);
        const int32_t asked = a.r.prompt ? a.r.prompt[s] : 0;
        const uint32_t answers = h0 + min(asked < 0 ? 0u : uint32_t(asked), h1 - h0);
        for (uint32_t i = h0 + tid; i < h1; i += kThreads) {
            const uint32_t t = uint32_t(a.r.history[i]) - lo;
            if (t < n) {
                if (i < answers)
                    atomicOr(counts + t, kSeen);
                else
                    atomicAdd(counts + t, 1u);
            }
        }
    }
    if (biased) {
        // each wave has a quarter of the chunk, and adds the biases there one after the other
        const uint32_t part = a.chunk / kWaves, p0 = lo + wave * part;
        for (uint32_t i0 = b0; i0 < b1; i0 += 64) {
            const uint32_t i = i0 + lane;
            const uint32_t t = i < b1 ? uint32_t(a.r.bias_token[i]) - p0 : part;
            const float v = i < b1 ? a.r.bias_value[i] : 0.0f;
            for (uint64_t m = __ballot(t < part && t + p0 < a.vocab); m != 0; m &= m - 1) {
                const int l = __builtin_ctzll(m);
                const uint32_t at = wave * part + __builtin_amdgcn_readlane(t, l);
                const float add = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l));
                if (lane == 0) bias[at] += add;
            }
        }
    }
    __syncthreads();
    for (; row < end; ++row) {
        if (counted && a.tokens) {
            const uint32_t t = uint32_t(a.tokens[row]) - lo;
            if (tid == 0 && t < n) counts[t] += 1;
            __syncthreads();
        }
        const uint32_t *mask = nullptr;
        if (a.r.mask) {
            const uint32_t m = a.r.mask_of ? uint32_t(a.r.mask_of[row]) : row;
            if (m < a.r.n_masks) mask = a.r.mask + size_t(m) * a.r.mask_words + (lo >> 5);
        }
        const uint64_t from = row * a.x_stride + lo, to = row * a.out_stride + lo;
        for (uint32_t i = tid * 4; i < n; i += kThreads * 4) {
            float l[4];
            const bool whole = i + 4 <= n;
            if (a.xtype == kF32) {
                const float *p = static_cast<const float *>(a.logits) + from + i;
                if (whole) {
                    const f32x4u v = *reinterpret_cast<const f32x4u *>(p);
#pragma unroll
                    for (int j = 0; j < 4; ++j) l[j] = v[j];
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) l[j] = i + j < n ? p[j] : 0.0f;
                }
            } else {
                const uint16_t *p = static_cast<const uint16_t *>(a.logits) + from + i;
                if (whole) {
                    const u16x4u v = *reinterpret_cast<const u16x4u *>(p);
#pragma unroll
                    for (int j = 0; j < 4; ++j) l[j] = widened(a.xtype, v[j]);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) l[j] = i + j < n ? widened(a.xtype, p[j]) : 0.0f;
                }
            }
            uint32_t allowed = 15;
            if (mask) allowed = mask[i >> 5] >> (i & 31);
            u32x4 c = {0, 0, 0, 0};
            f32x4 b = {0.0f, 0.0f, 0.0f, 0.0f};
            if (counted) c = *reinterpret_cast<const u32x4 *>(counts + i);
            if (biased) b = *reinterpret_cast<const f32x4 *>(bias + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (c[j] != 0 || b[j] != 0.0f) l[j] = changed(l[j], c[j], b[j], rep, freq, pres);
                if (!(allowed >> j & 1)) l[j] = -kInf;
            }
            float *o = a.out + to + i;
            if (whole) {
                *reinterpret_cast<f32x4u *>(o) = f32x4u{l[0], l[1], l[2], l[3]};
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (i + j < n) o[j] = l[j];
            }
        }
        if (counted && a.tokens) __syncthreads();
    }
}

}  // namespace

hipError_t launch_logits(LogitCall c, int num_cu, hipStream_t st) {
    // chunks of 1024 to 8192 tokens, as many as make about 8 workgroups per CU
    const uint64_t want = std::max<uint64_t>(1, uint64_t(c.vocab) * c.n_seq / (8 * uint64_t(num_cu)));
    c.chunk = want > 4096 ? 8192 : want > 2048 ? 4096 : want > 1024 ? 2048 : 1024;
    const uint32_t bytes = c.chunk * (c.r.bias_start ? 8 : 4);
    k_logits<<<dim3((c.vocab + c.chunk - 1) / c.chunk, c.n_seq), kThreads, bytes, st>>>(c);
    return hipGetLastError();
}

}  // namespace tc
