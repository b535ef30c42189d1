// tc_attn_common.hpp -- what the paged-cache kernels share: the batch as the
// kernels see it, element types and their conversions, and the launchers.
#pragma once

#include "tc_common.hpp"

namespace tc {

// Element types of rows and caches (tc_attention.h).
enum : int { kF32 = 0, kF16 = 1, kI8 = 24, kBF16 = 30, kE4M3 = 100 };

__host__ __device__ constexpr uint32_t elem_bytes(int t) { return t == kF32 ? 4 : t == kF16 || t == kBF16 ? 2 : 1; }
__host__ __device__ constexpr bool scaled_type(int t) { return t == kI8 || t == kE4M3; }

constexpr uint32_t kMaxHeadDim = 256;

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// Two bf16 of two floats, to nearest even (NaN stays NaN).
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    return __builtin_bit_cast(uint32_t, bf16x2{__bf16(a), __bf16(b)});
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    return __builtin_bit_cast(uint32_t, f16x2{_Float16(a), _Float16(b)});
}

// 8 consecutive elements of a row as floats (16-byte aligned rows).
__device__ __forceinline__ void load8(int type, const void *p, uint64_t elem, float (&x)[8]) {
    if (type == kF32) {
        const f32x4 *q = reinterpret_cast<const f32x4 *>(static_cast<const float *>(p) + elem);
        const f32x4 u = q[0], v = q[1];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = u[i], x[4 + i] = v[i];
    } else {
        const u32x4 u = *reinterpret_cast<const u32x4 *>(static_cast<const uint16_t *>(p) + elem);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = u[i];
            if (type == kF16) {
                x[2 * i] = h2f(w & 0xFFFF);
                x[2 * i + 1] = h2f(w >> 16);
            } else {
                x[2 * i] = __builtin_bit_cast(float, w << 16);
                x[2 * i + 1] = __builtin_bit_cast(float, w & 0xFFFF0000u);
            }
        }
    }
}

__device__ __forceinline__ void store8(int type, void *p, uint64_t elem, const float (&x)[8]) {
    if (type == kF32) {
        f32x4 *q = reinterpret_cast<f32x4 *>(static_cast<float *>(p) + elem);
        q[0] = f32x4{x[0], x[1], x[2], x[3]};
        q[1] = f32x4{x[4], x[5], x[6], x[7]};
    } else {
        u32x4 u;
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = type == kF16 ? pack_f16(x[2 * i], x[2 * i + 1]) : pack_bf16(x[2 * i], x[2 * i + 1]);
        *reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(p) + elem) = u;
    }
}

// ---- launchers (tc_kv.hip, tc_attn.hip, tc_verify.hip) ----
hipError_t launch_kv_write(const KvArgs &a, int ctype, int xtype, const void *k, const void *v, uint32_t k_stride,
                           uint32_t v_stride, hipStream_t st);
hipError_t launch_kv_read(const KvArgs &a, int ctype, int xtype, void *k, void *v, hipStream_t st);

// As find_seq, 64 sequences at a time: one fetch where there are no more. The first 64 may be
// fetched ahead.
struct SeqProbe {
    int32_t start;
};
__device__ __forceinline__ SeqProbe probe_seqs(const int32_t *start, uint32_t n_seq) {
    return {start[min((threadIdx.x & 63) * ((n_seq + 63) / 64), n_seq)]};
}
__device__ __forceinline__ int wave_find_seq(const int32_t *start, uint32_t n_seq, uint32_t t, SeqProbe probe) {
    const uint32_t lane = threadIdx.x & 63;
    const int32_t before = start[0], behind = start[n_seq];
    uint32_t lo = 0, hi = n_seq;
    for (int32_t v = probe.start; hi - lo > 1;) {
        const uint32_t step = (hi - lo + 63) / 64, p = lo + lane * step;
        const uint64_t m = __ballot(p < hi && (p == lo || v <= int32_t(t)));
        lo += (63 - __builtin_clzll(m)) * step;
        hi = min(lo + step, hi);
        if (hi - lo > 1) v = start[min(lo + lane * ((hi - lo + 63) / 64), n_seq)];
    }
    return int32_t(t) >= behind || int32_t(t) < before ? -1 : int(lo);
}
__device__ __forceinline__ int wave_find_seq(const int32_t *start, uint32_t n_seq, uint32_t t) {
    return wave_find_seq(start, n_seq, t, probe_seqs(start, n_seq));
}

struct AttnArgs {
    KvArgs kv;
    const void *q;
    void *out;
    uint32_t heads, group;  // query heads, query heads per key/value head
    DivMod group_div;
    uint32_t q_stride;
    float scale;
    int32_t cap;   // tokens that the table has room for
    int32_t span;  // tokens that a row sees at most: the window
    int xtype;
};
size_t attn_scratch_bytes(int num_cu);
hipError_t launch_attn(const AttnArgs &a, int ctype, int num_cu, void *scratch, hipStream_t st);
// ... for one cache type (tc_attn_inst.hip).
template <int CT>
hipError_t launch_attn_cache(const AttnArgs &a, int num_cu, void *scratch, hipStream_t st);
template <>
hipError_t launch_attn_cache<kF16>(const AttnArgs &a, int num_cu, void *scratch, hipStream_t st);
template <>
hipError_t launch_attn_cache<kBF16>(const AttnArgs &a, int num_cu, void *scratch, hipStream_t st);
template <>
hipError_t launch_attn_cache<kI8>(const AttnArgs &a, int num_cu, void *scratch, hipStream_t st);
template <>
hipError_t launch_attn_cache<kE4M3>(const AttnArgs &a, int num_cu, void *scratch, hipStream_t st);

// A block of rows whose tiles lie in several parts.
struct SplitJob {
    uint32_t begin, r0, kvh;  // the sequence's first token row; the block's first row
    uint32_t rows;   // of the block
    uint32_t count;  // parts, from this one on (0: none)
    uint32_t slot;   // where the first one's sums are; the others': 2 * part
};

// Sums that workgroups leave for k_attn_join: two blocks of rows each, in slots of as
// many rows as the larger kind of block has.
struct SplitScratch {
    SplitJob *jobs;  // [parts]
    float *ml;       // [2 * parts][rows][2] reference and sum of weights
    float *o;        // [2 * parts][rows][DP] sums
};
inline SplitScratch split_scratch(void *scratch, uint32_t parts, uint32_t rows) {
    char *p = static_cast<char *>(scratch);
    SplitScratch s;
    s.jobs = reinterpret_cast<SplitJob *>(p);
    p += (parts * sizeof(SplitJob) + 255) & ~size_t(255);
    s.ml = reinterpret_cast<float *>(p);
    p += size_t(parts) * 2 * rows * 2 * 4;
    s.o = reinterpret_cast<float *>(p);
    return s;
}
// Sequences of at most this many rows (new tokens * query heads per key/value
// head) are served in blocks of 16, the others in blocks of 128 or 256.
constexpr uint32_t kFewRows = 64;
// For any call: a part per CU, with slots of 256 rows of up to 128 dims or 128 of up
// to 256.
inline size_t attn_part_bytes(int num_cu) {
    const size_t cu = num_cu, jobs = (cu * sizeof(SplitJob) + 255) & ~size_t(255);
    return jobs + cu * 2 * 256 * 2 * 4 + cu * 2 * 256 * 128 * 4;
}

struct VerifyArgs {
    const float *logits, *draft_probs;
    uint32_t vocab, n_seq, n_tokens;
    const int32_t *start, *tokens;
    const float *temperature, *accept_u, *sample_u;
    int32_t *n_accepted, *next_token;
};
size_t verify_scratch_bytes(uint32_t n_tokens, uint32_t n_seq);
hipError_t launch_verify(const VerifyArgs &a, int num_cu, void *scratch, hipStream_t st);

}  // namespace tc
