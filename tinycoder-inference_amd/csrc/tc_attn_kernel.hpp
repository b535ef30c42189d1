// tc_attn_kernel.hpp -- causal attention of a chunk of new tokens over a paged
// cache: the parts that its kernels share.
//
// The mathematics. For a key/value head, rows r = (new token, query head of its
// group) and cached tokens j, with t_rj = log2(e) * scale * q_r . k_j:
//   o_r = sum_j 2^(t_rj - m_r) v_j / sum_j 2^(t_rj - m_r)
// for any reference m_r, so one pass over the cache does, with m_r raised (and the
// sums so far multiplied) only where a score exceeds it by 2^kLazy.
//
// On the matrix cores, 32 rows at a time as columns: scores = K Q^T (tokens by
// rows, v_mfma_f32_32x32x16), o^T += V^T P^T (dims by rows). A lane then holds one
// row's scores of 16 tokens and the same row's sums, so maxima, exponentials and
// the raising of m need one exchange between the wave's halves and no other. The
// scores come out of the first product in the registers in which the second one
// takes them, if the tokens are numbered 16 (i / 8) + 8 half + i % 8 for register
// i: the first product's operand rows are read in that order (token_of_row). V is
// stored by rows and enters by columns: ds_read_b64_tr_b16 / _b8 transpose on the
// way out of LDS.
//
// Operands: F16 and the 8-bit caches as fp16 (both exact there), BF16 as bf16. Rows
// and weights of more bits go as several pieces, each exact product accumulated in
// fp32. Rows bound for fp16 are first scaled by a power of two to a largest value
// in [2^14, 2^15); weights carry a factor 2^kLift, which keeps those that matter
// out of fp16's subnormals and cancels in the quotient. A factor per token (8-bit
// caches): the key's multiplies the score; the value's goes into the weight as
// 2^(t + log2 v_scale - m), and the sum of weights takes it out again.
#pragma once

#include "tc_attn_common.hpp"
#include "tc_kernels.hpp"

namespace tc {
namespace {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int s32x2 __attribute__((ext_vector_type(2)));
typedef int s32x4 __attribute__((ext_vector_type(4)));

constexpr float kLazy = 4.0f, kLift = 11.0f;
constexpr uint32_t kTileTokens = 32;  // tokens of one score product
constexpr float kNegInf = -__builtin_inff();

// ---- LDS tiles --------------------------------------------------------------
// Rows of RB bytes in 16-byte chunks, chunk c of row r at place c ^ swizzle(r), so
// that the lanes of one LDS cycle (256 bytes) fall on different banks: 16
// consecutive rows of one chunk (keys, rows of q), or 4 (16-bit) or 8 (8-bit)
// consecutive rows of 64 or 32 bytes each (values, read transposed).
template <int RB>
__device__ __forceinline__ constexpr uint32_t key_swizzle(uint32_t r) {
    return RB >= 256 ? r & 15 : (r / (256 / RB)) & (RB / 16 - 1);
}
template <int RB, int ES>
__device__ __forceinline__ constexpr uint32_t value_swizzle(uint32_t r) {
    constexpr uint32_t rp = RB >= 256 ? 1 : 256 / RB, rows = ES == 2 ? 4 : 8, cw = ES == 2 ? 4 : 2;
    return cw * ((r / rp) & (rows / rp - 1));
}

__device__ __forceinline__ uint32_t lds_addr(const void *p) {
    return uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const void *)(p)));
}

// Lane l's 16 (4) bytes at base + off to LDS byte dst + 16 l (4 l), asynchronously:
// the kernel waits (vmcnt) before it reads them. Inline, so that the compiler does
// not wait for these at every LDS read in between; m0 is restored.
__device__ __forceinline__ void dma16(uint32_t dst, const void *base, uint32_t off) {
    uint32_t saved;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %2, %3\n\ts_mov_b32 m0, %0"
                 : "=&s"(saved)
                 : "s"(__builtin_amdgcn_readfirstlane(dst)), "v"(off), "s"(base)
                 : "memory");
}
__device__ __forceinline__ void dma4(uint32_t dst, const void *base, uint32_t off) {
    uint32_t saved;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\tglobal_load_lds_dword %2, %3\n\ts_mov_b32 m0, %0"
                 : "=&s"(saved)
                 : "s"(__builtin_amdgcn_readfirstlane(dst)), "v"(off), "s"(base)
                 : "memory");
}
template <int N>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// (before a load overwrites what LDS reads in flight may still fetch)
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// ---- operands ---------------------------------------------------------------

template <int CT>
__device__ __forceinline__ v16f mfma(u32x4 a, u32x4 b, v16f c) {
    if constexpr (CT == kBF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// 4 cache bytes as 4 fp16, exactly. I8: b ^ 0x80 under the exponent of 1024 is
// 1152 + b.
template <int CT>
__device__ __forceinline__ u32x2 widen(uint32_t w) {
    if constexpr (CT == kI8) {
        const uint32_t u = w ^ 0x80808080u;
        const f16x2 off = {_Float16(1152.0f), _Float16(1152.0f)};
        const f16x2 lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - off;
        const f16x2 hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - off;
        return u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
    } else {
        const auto lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(int(w), 1.0f, false);
        const auto hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(int(w), 1.0f, true);
        return u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
    }
}

// The token (of 32) whose key is row m of the first product.
__device__ __forceinline__ uint32_t token_of_row(uint32_t m) { return (m & 19) | ((m & 4) << 1) | ((m & 8) >> 1); }
// The token of score register i in a half of the wave.
__device__ __forceinline__ uint32_t token_of_reg(uint32_t i, uint32_t half) { return 16 * (i / 8) + 8 * half + i % 8; }

// First of the 8 dims of contraction step ks in a half of the wave: 16-bit rows
// are read in 16-byte chunks of 8 dims, 8-bit ones in chunks of 16, for two steps.
template <int ES>
__device__ __forceinline__ uint32_t step_dim(uint32_t ks, uint32_t half) {
    return ES == 2 ? 16 * ks + 8 * half : 32 * (ks / 2) + 16 * half + 8 * (ks % 2);
}

// One or more 16-bit pieces of x: x = sum of the pieces but for what is below them.
template <int CT>
__device__ __forceinline__ uint32_t piece2(float &a, float &b) {
    if constexpr (CT == kBF16) {
        const uint32_t w = pack_bf16(a, b);
        a -= __builtin_bit_cast(float, w << 16);
        b -= __builtin_bit_cast(float, w & 0xFFFF0000u);
        return w;
    } else {
        const f16x2 h = {_Float16(a), _Float16(b)};
        a -= float(h[0]);
        b -= float(h[1]);
        return __builtin_bit_cast(uint32_t, h);
    }
}

// Largest magnitude's exponent e such that x * 2^-e is in [2^14, 2^15) for fp16
// operands; 0 for bf16 ones, zeros and rows that are not finite.
template <int CT>
__device__ __forceinline__ int row_exponent(float m) {
    if (CT == kBF16 || !(m > 0.0f) || m == __builtin_inff()) return 0;
    return __builtin_amdgcn_frexp_expf(m) - 15;
}

// Values that are not finite in four cache bytes.
template <int CT>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
    if constexpr (CT == kF16) return ((w & 0x7C007C00u) + 0x04000400u) & 0x80008000u;
    if constexpr (CT == kBF16) return ((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u;
    if constexpr (CT == kE4M3) return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
    return 0;
}

// Four consecutive cache elements as floats.
template <int CT>
__device__ __forceinline__ void value4(const unsigned char *p, float (&x)[4]) {
    if constexpr (scaled_type(CT)) {
        const u32x2 h = widen<CT>(*reinterpret_cast<const uint32_t *>(p));
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = h2f(i & 1 ? h[i / 2] >> 16 : h[i / 2] & 0xFFFF);
    } else {
        const u32x2 w = *reinterpret_cast<const u32x2 *>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t b = i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xFFFF;
            x[i] = CT == kF16 ? h2f(b) : __builtin_bit_cast(float, b << 16);
        }
    }
}

// Output dims e .. e + 3 (or e alone) of a row of a sequence's block.
__device__ __forceinline__ uint64_t out_at(const AttnArgs &a, uint32_t begin, uint32_t kvh, uint32_t row) {
    const uint32_t tok = row / a.group;
    return (uint64_t(begin + tok) * a.heads + kvh * a.group + row - tok * a.group) * a.kv.dim;
}
__device__ __forceinline__ void store4(const AttnArgs &a, uint32_t begin, uint32_t kvh, uint32_t row, uint32_t e, f32x4 x) {
    const uint64_t at = out_at(a, begin, kvh, row) + e;
    if (a.xtype == kF32) {
        *reinterpret_cast<f32x4 *>(static_cast<float *>(a.out) + at) = x;
    } else {
        const u32x2 w = a.xtype == kF16 ? u32x2{pack_f16(x[0], x[1]), pack_f16(x[2], x[3])}
                                        : u32x2{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])};
        *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(a.out) + at) = w;
    }
}
__device__ __forceinline__ void store1(const AttnArgs &a, uint32_t begin, uint32_t kvh, uint32_t row, uint32_t e, float x) {
    const uint64_t at = out_at(a, begin, kvh, row) + e;
    if (a.xtype == kF32)
        static_cast<float *>(a.out)[at] = x;
    else
        static_cast<uint16_t *>(a.out)[at] = uint16_t(a.xtype == kF16 ? pack_f16(x, x) : pack_bf16(x, x));
}

// v of the lane 32 away.
__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32); }

// ---- rows of q --------------------------------------------------------------
// 32 rows of NP pieces in LDS, [NP][32][DP] 16-bit elements in swizzled chunks, and
// each row's factor log2(e) * scale * 2^e. Row r is query head (r0 + r) % group of
// token row (r0 + r) / group; rows at n_rows or above are zeros. THREADS threads.
template <int CT, int NP, int DP, int THREADS>
__device__ __forceinline__ void stage_q(const AttnArgs &a, uint32_t begin, uint32_t kvh, uint32_t r0, uint32_t n_rows,
                                        unsigned char *lds, float *factor, uint32_t tid) {
    constexpr uint32_t QB = 2 * DP, per = THREADS / 32, chunks = DP / 8;
    static_assert(chunks % per == 0, "");
    const uint32_t r = tid / per, l = tid % per, row = r0 + r;
    const uint32_t tok = row / a.group;
    const uint64_t at = uint64_t(begin + tok) * a.q_stride + uint64_t(kvh * a.group + row - tok * a.group) * a.kv.dim;
    float x[chunks / per][8];
    float m = 0.0f;
#pragma unroll
    for (uint32_t k = 0; k < chunks / per; ++k) {
        const uint32_t d = 8 * (l + per * k);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[k][i] = 0.0f;
        if (row < n_rows && d < a.kv.dim) load8(a.xtype, a.q, at + d, x[k]);
#pragma unroll
        for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(x[k][i]));
    }
#pragma unroll
    for (uint32_t o = 1; o < per; o <<= 1) m = fmaxf(m, __shfl_xor(m, int(o)));
    const int e = row_exponent<CT>(m);
#pragma unroll
    for (uint32_t k = 0; k < chunks / per; ++k) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[k][i] = ldexpf(x[k][i], -e);
        const uint32_t c = l + per * k;
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            u32x4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = piece2<CT>(x[k][2 * i], x[k][2 * i + 1]);
            *reinterpret_cast<u32x4 *>(lds + (p * 32 + r) * QB + ((c ^ key_swizzle<QB>(r)) << 4)) = w;
        }
    }
    if (l == 0) factor[r] = ldexpf(1.4426950408889634f * a.scale, e);
}

}  // namespace
}  // namespace tc
