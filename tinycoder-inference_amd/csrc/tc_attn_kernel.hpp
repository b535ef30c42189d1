// tc_attn_kernel.hpp -- causal attention of a chunk of new tokens over a paged
// cache: the parts that its kernels share.
//
// The mathematics. For a key/value head, rows r = (new token, query head of its
// group) and cached tokens j, with t_rj = log2(e) * scale * q_r . k_j:
//   o_r = sum_j 2^(t_rj - m_r) v_j / sum_j 2^(t_rj - m_r)
// for any reference m_r, so one pass over the cache does, with m_r raised (and the
// sums so far multiplied) only where a score exceeds it by 2^kLazy.
//
// On the matrix cores, R = 16 or 32 rows at a time as columns: scores = K Q^T (tokens
// by rows), o^T += V^T P^T (dims by rows), v_mfma_f32_16x16x32 or _32x32x16. A lane
// then holds scores of one row (its column, lane % R) and the same row's sums;
// maxima and sums over a row's lanes, one in each of the 64 / R groups, take an
// exchange or two. The scores come out of the first product in the registers in
// which the second one takes them, if score register i of group g is the token
// token_of_reg(i, g): the first product's operand rows are read in that order. V is
// stored by rows and enters by columns: ds_read_b64_tr_b16 / _b8 transpose on the way
// out of LDS. 32 rows halve the LDS reads per product, 16 the registers of the sums
// and of q, and the work where there are no more rows.
//
// Operands: F16 and the 8-bit caches as fp16 (both exact there), BF16 as bf16. Rows
// and weights of more bits go as several pieces, each exact product accumulated in
// fp32. Rows bound for fp16 are first scaled by a power of two to a largest value
// in [2^14, 2^15); weights carry a factor 2^kLift, which keeps those that matter
// out of fp16's subnormals and cancels in the quotient. A factor per token (8-bit
// caches): the key's multiplies the score; the value's goes into the weight as
// 2^(t + log2 v_scale - m), and the sum of weights takes it out again (value_factor).
#pragma once

#include "tc_attn_common.hpp"
#include "tc_kernels.hpp"

namespace tc {
namespace {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int s32x2 __attribute__((ext_vector_type(2)));

constexpr float kLazy = 4.0f, kLift = 11.0f;
constexpr uint32_t kTileTokens = 32;
constexpr float kNegInf = -__builtin_inff();

// Shapes of the products for R rows and a padded head size.
template <int R, int DP>
struct Geo {
    static constexpr int G = 64 / R;                // groups of lanes
    static constexpr int NS = R / 2;                // scores of a lane: 32 tokens by R rows
    static constexpr int AE = R == 32 ? 16 : 4;     // registers of an accumulator
    static constexpr int NA = NS / AE;              // score accumulators
    static constexpr int KS = DP * R / 512;         // contraction steps over the dims: 16 or 32 each
    static constexpr int KT = R == 32 ? 2 : 1;      // ... over the tokens: 16 or 32 each
    static constexpr int DB = DP / R;               // blocks of R dims
};
template <int R>
struct AccOf {
    typedef v16f type;
};
template <>
struct AccOf<16> {
    typedef f32x4 type;
};
template <int R>
using Acc = typename AccOf<R>::type;

// The lane's index recomputed where it is used (v_mbcnt on an opaque zero): what rare
// paths derive from it is then not held in registers across the loops.
__device__ __forceinline__ uint32_t lane_now() {
    uint32_t z = 0;
    asm volatile("" : "+s"(z));
    return __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, z));
}

// ---- LDS tiles --------------------------------------------------------------
// Rows of RB bytes in 16-byte chunks, chunk c of row r at place c ^ swizzle(r), so
// that the lanes of one LDS cycle (256 bytes) fall on different banks. Keys: 16
// lanes read one chunk of as many rows, consecutive ones (R = 32), or four runs of
// four, 8 apart (R = 16). Values, read transposed by 32 lanes: R = 32: 64 bytes of 4
// consecutive rows; R = 16: 32 bytes of two such runs, 8 apart (8-bit: 16 bytes of 16
// consecutive rows).
template <int R, int RB>
__device__ __forceinline__ constexpr uint32_t key_swizzle(uint32_t r) {
    const uint32_t x = R == 32 ? r & 15 : (r & 3) | ((r >> 1) & 12);  // 16 rows told apart
    return RB >= 256 ? x : (x / (256 / RB)) & (RB / 16 - 1);
}
template <int R, int RB, int ES>
__device__ __forceinline__ constexpr uint32_t value_swizzle(uint32_t r) {
    constexpr uint32_t rp = RB >= 256 ? 1 : 256 / RB;  // rows of one LDS cycle
    if (ES == 1) return (r / rp) & (16 / rp - 1);
    const uint32_t x = R == 32 ? r & 3 : (r & 3) | ((r >> 1) & 4);
    return (R == 32 ? 4 : 2) * ((x / rp) & ((R == 32 ? 4 : 8) / rp - 1));
}

__device__ __forceinline__ uint32_t lds_addr(const void *p) {
    return uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const void *)(p)));
}

// Lane l's 16 (4) bytes to LDS byte dst + 16 l (4 l), asynchronously:
// the kernel waits (vmcnt) before it reads them. Inline, so that the compiler does
// not wait for these at every LDS read in between; m0 (the LDS address) is restored:
// the compiler may hold a value there. The s_nop: a load takes an LDS address one wait
// state after a scalar write of m0, and a scalar operand five after a vector instruction
// (readfirstlane) wrote it; the compiler counts neither for inline code. ONCE: the line is not read again soon.
template <bool ONCE = false>
__device__ __forceinline__ void dma16(uint32_t dst, const void *base, uint32_t off) {
    const uint64_t b = reinterpret_cast<uint64_t>(base);
    // (readfirstlane gives an int: widened as one, its sign would fill the upper half)
    const uint32_t blo = __builtin_amdgcn_readfirstlane(uint32_t(b)), bhi = __builtin_amdgcn_readfirstlane(uint32_t(b >> 32));
    const uint64_t ub = uint64_t(bhi) << 32 | blo;
    uint32_t saved;
    if constexpr (ONCE)
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 2\n\tglobal_load_lds_dwordx4 %2, %3 nt\n\ts_mov_b32 m0, %0"
                     : "=&s"(saved)
                     : "s"(__builtin_amdgcn_readfirstlane(dst)), "v"(off), "s"(ub)
                     : "memory");
    else
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 2\n\tglobal_load_lds_dwordx4 %2, %3\n\ts_mov_b32 m0, %0"
                     : "=&s"(saved)
                     : "s"(__builtin_amdgcn_readfirstlane(dst)), "v"(off), "s"(ub)
                     : "memory");
}
__device__ __forceinline__ void dma4(uint32_t dst, const void *p) {  // (4 bytes of each lane's own)
    uint32_t saved;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 2\n\tglobal_load_lds_dword %2, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(saved)
                 : "s"(__builtin_amdgcn_readfirstlane(dst)), "v"(p)
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
template <int CT>
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (CT == kBF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Keeps a product where it stands among what follows (nothing is emitted): the
// accumulator counts as changed here.
template <class T>
__device__ __forceinline__ void pin(T &acc) {
    asm volatile("" : "+v"(acc));
}

// A value that the compiler cannot form ahead of this point, nor hold what it would
// form from it in registers of the paths around.
__device__ __forceinline__ uint32_t here(uint32_t v) {
    asm volatile("" : "+v"(v));
    return v;
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

// The token (of 32) whose key is operand row m of score accumulator a.
template <int R>
__device__ __forceinline__ uint32_t token_of_row(uint32_t m, uint32_t a) {
    return R == 32 ? (m & 19) | ((m & 4) << 1) | ((m & 8) >> 1) : 8 * (m / 4) + 4 * a + m % 4;
}
// The token of score register i in group g.
template <int R>
__device__ __forceinline__ uint32_t token_of_reg(uint32_t i, uint32_t g) {
    return R == 32 ? 16 * (i / 8) + 8 * g + i % 8 : 8 * g + i;
}
// The dims of quad k (registers 4 k to 4 k + 3) of a block of R dims in group g.
__device__ __forceinline__ uint32_t dim_of_quad(uint32_t k, uint32_t g) { return 8 * k + 4 * g; }

// First of the 8 dims of contraction step ks in group g: 16-bit rows are read in
// 16-byte chunks of 8 dims, 8-bit ones in chunks of 16, for two steps.
template <int R, int ES>
__device__ __forceinline__ uint32_t step_dim(uint32_t ks, uint32_t g) {
    constexpr uint32_t G = 64 / R;
    return ES == 2 ? 8 * (G * ks + g) : 16 * (G * (ks / 2) + g) + 8 * (ks % 2);
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

// Over a row's lanes, one in each group; the result in all of them.
template <int R, class F>
__device__ __forceinline__ float over_groups(float v, F f) {
    uint32_t b = __builtin_bit_cast(uint32_t, v);
    const auto h = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    v = f(__builtin_bit_cast(float, uint32_t(h[0])), __builtin_bit_cast(float, uint32_t(h[1])));
    if constexpr (R == 16) {
        b = __builtin_bit_cast(uint32_t, v);
        const auto q = __builtin_amdgcn_permlane16_swap(b, b, false, false);
        v = f(__builtin_bit_cast(float, uint32_t(q[0])), __builtin_bit_cast(float, uint32_t(q[1])));
    }
    return v;
}
template <int R>
__device__ __forceinline__ float groups_max(float v) {
    return over_groups<R>(v, [](float a, float b) { return fmaxf(a, b); });
}
template <int R>
__device__ __forceinline__ float groups_sum(float v) {
    return over_groups<R>(v, [](float a, float b) { return a + b; });
}

// (maximum, which keeps NaN, is one instruction for three; fmaxf would first quiet its
// operands, an instruction each)
__device__ __forceinline__ float max3(float a, float b, float c) {
    return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}
// a.x * b.x + a.y * b.y + c of 16-bit pairs; b is two ones: the sum of two weights as
// they enter the products.
template <int CT>
__device__ __forceinline__ float add_pair(uint32_t w, float c) {
    if constexpr (CT == kBF16) {
        const bf16x2 one = {__bf16(1.0f), __bf16(1.0f)};
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), one, c, false);
    } else {
        const f16x2 one = {_Float16(1.0f), _Float16(1.0f)};
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w), one, c, false);
    }
}

// Whether the sum of weights is that of the weights as they enter the products. One piece of
// 16 bits is off by up to half a step, in the sums of values and in that of the weights alike,
// and the quotient keeps less of it (values that are all alike come out as they are). More
// pieces hold what fp32 rows ask for. Not with factors: there a token whose values are nothing
// has a weight below its piece's least, and counts in the sum all the same.
template <int CT, int NP>
__device__ constexpr bool rounded_sum() { return NP == 1 && !scaled_type(CT); }

template <int N>
__device__ __forceinline__ float max_of(const float (&x)[N]) {
    float m = max3(x[0], x[1], x[2]), n = max3(x[3], x[4], x[5]);
#pragma unroll
    for (int i = 6; i + 3 < N; i += 4) m = max3(m, x[i], x[i + 1]), n = max3(n, x[i + 2], x[i + 3]);
    return max3(m, max3(n, x[N - 2], x[N - 1]), n);
}

// A value's factor as weights take it: at least 2^kLeast (NaN stays). A token whose values
// are nothing, by a factor of 0 as in a slot that was never written, or next to it, still
// has its weight, 2^(t + log2 factor - m + kLift) divided by the factor, in the sum of
// weights: from 2^-80 on neither is the one lost below 2^-126 (nor the products that raise m)
// where it is 2^-24 of the largest beside factors of up to 2^22, nor do 2^31 of the other, up
// to 2^95 each, pass fp32's end.
constexpr float kLeast = -80.0f;
__device__ __forceinline__ float value_factor(float x) { return x == x ? fmaxf(x, 0x1p-80f) : x; }

// tc_kv_write gives a row of zeros the factor 1. Beside values of 1e-6 that would put m 2^27
// above what the others' weights reach, and their pieces would lose as many bits; so rows of
// factor 1 are looked at, and those of zeros count as of factor 2^kLeast. Most show in their
// first values that they are not, so that caches whose factors are all 1 take 0 to 7% longer
// (17 to 65% where whole rows were read; 1% where no factor is 1).
template <int CT>
__device__ __forceinline__ bool zeros16(u32x4 w) {  // (an 8-bit float's zero has a sign)
    return ((w[0] | w[1] | w[2] | w[3]) & (CT == kE4M3 ? 0x7F7F7F7Fu : ~0u)) == 0;
}
template <int CT>
__device__ __forceinline__ bool row_of_zeros(const uint8_t *row, uint32_t rowbytes) {
    bool z = true;
#pragma unroll 1
    for (uint32_t i = 0; i < rowbytes && z; i += 16) z = zeros16<CT>(*reinterpret_cast<const u32x4 *>(row + i));
    return z;
}
// For few rows the values are on their way to LDS when their factors are wanted, so there the
// look is taken where m rises, and only there: which of a tile's 32 rows, of those whose bits are set, are zeros.
template <int CT, int RB>
__device__ __forceinline__ uint32_t rows_of_zeros(uint32_t may, const unsigned char *vt, uint32_t lane) {
    const unsigned char *half = vt + lane % 32 * RB + lane / 32 * (RB / 2);
#pragma unroll 1
    for (uint32_t i = 0; i < RB / 2 && may != 0; i += 16) {
        const uint64_t z = __ballot(zeros16<CT>(*reinterpret_cast<const u32x4 *>(half + i)));
        may &= uint32_t(z) & uint32_t(z >> 32);
    }
    return may;
}
// Their scores as exponents of that factor, before m is chosen; ...
template <int R, int NS>
__device__ __forceinline__ void lower_zeros(float (&s)[NS], uint32_t zeros, uint32_t g) {
#pragma unroll
    for (int i = 0; i < NS; ++i)
        if ((zeros >> token_of_reg<R>(i, g)) & 1) s[i] += kLeast;
}
// ... behind that, their weights' sum, taken out of the scores.
template <int R, int NS>
__device__ __forceinline__ float take_zeros(float (&s)[NS], uint32_t zeros, uint32_t g, float ref) {
    float l = 0.0f;
#pragma unroll
    for (int i = 0; i < NS; ++i)
        if ((zeros >> token_of_reg<R>(i, g)) & 1) {
            l = fmaf(__builtin_amdgcn_exp2f(s[i] - ref), 0x1p80f, l);
            s[i] = kNegInf;
        }
    return l;
}

// 16 bytes of LDS at an address of lds_addr's.
typedef const __attribute__((address_space(3))) u32x4 *lds_u32x4;
__device__ __forceinline__ u32x4 lds_at(uint32_t addr) { return *reinterpret_cast<lds_u32x4>(addr); }
__device__ __forceinline__ u32x2 lds_transposed16(uint32_t addr) {
    return __builtin_bit_cast(u32x2,
                              __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<__attribute__((address_space(3))) s16x4 *>(addr)));
}

// Operands from 16-bit tiles at LDS addresses. Scores: the lane's place for
// accumulator a and step 0, which step ks changes by an exclusive or (the step's
// chunk number and the group's share no bits).
template <int R, int RB>
__device__ __forceinline__ uint32_t key_place(uint32_t a, uint32_t lane) {
    const uint32_t r = token_of_row<R>(lane % R, a);
    return r * RB + (((lane / R) ^ key_swizzle<R, RB>(r)) << 4);
}
template <int R>
__device__ __forceinline__ uint32_t key_step(uint32_t ks) {
    return ks * (64 / R) * 16;
}
// Values: the lane's place for dims 0 to R - 1, which block d changes by an exclusive
// or; the rows of step k differ from those of step 0 in no bit that the swizzle takes.
template <int R, int RB>
__device__ __forceinline__ uint32_t value_place(uint32_t lane) {
    const uint32_t l16 = lane & 15, g = lane / R;
    const uint32_t r = 8 * g + l16 / 4, e = (lane % R) / 16 * 16 + 4 * (l16 % 4);
    return r * RB + (((e / 8) ^ value_swizzle<R, RB, 2>(r)) << 4) + (e & 4) * 2;
}
template <int R>
__device__ __forceinline__ uint32_t value_block(uint32_t d) {
    return 2 * R * d;
}
template <int RB>
__device__ __forceinline__ u32x4 value_frag(uint32_t vt_place, uint32_t k) {
    const u32x2 a = lds_transposed16(vt_place + 16 * k * RB), b = lds_transposed16(vt_place + (16 * k + 4) * RB);
    return u32x4{a[0], a[1], b[0], b[1]};
}

// Whether a tile in LDS holds a value that is not finite.
template <int CT, int TILE>
__device__ __forceinline__ bool tile_not_finite(const unsigned char *vt, uint32_t lane) {
    uint32_t bad = 0;
    for (uint32_t i = lane; i < TILE / 16; i += 64) {
        const u32x4 w = *reinterpret_cast<const u32x4 *>(vt + 16 * i);
        bad |= not_finite<CT>(w[0]) | not_finite<CT>(w[1]) | not_finite<CT>(w[2]) | not_finite<CT>(w[3]);
    }
    return __ballot(bad != 0) != 0;
}

// o += weights * values token by token, of those that the lane's row sees alone: for
// tiles with infinities or NaN that some row must not see, which a product with a
// weight of 0 would bring in.
template <int CT, int R, int RB, int DP>
__device__ __forceinline__ void add_values_one_by_one(const unsigned char *vt, const float (&s)[R / 2], uint32_t seen, uint32_t lane,
                                                      Acc<R> (&o)[DP / R]) {
    constexpr uint32_t ES = scaled_type(CT) ? 1 : 2, G = 64 / R;
    const uint32_t col = lane % R, g = lane / R;
    for (uint32_t i = 0; i < R / 2; ++i)
        for (uint32_t h = 0; h < G; ++h) {
            float p = 0.0f;
#pragma unroll
            for (int j = 0; j < R / 2; ++j) p = i == uint32_t(j) ? s[j] : p;
            const bool sees = (__shfl(seen, int(col + R * h)) >> i) & 1;
            p = __shfl(p, int(col + R * h));
            const uint32_t r = token_of_reg<R>(i, h);
#pragma unroll
            for (int d = 0; d < DP / R; ++d)
#pragma unroll
                for (int k = 0; k < (R == 32 ? 4 : 1); ++k) {
                    const uint32_t byte = (R * d + dim_of_quad(k, g)) * ES;
                    float x[4];
                    value4<CT>(vt + r * RB + (((byte / 16) ^ value_swizzle<R, RB, ES>(r)) << 4) + byte % 16, x);
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[d][4 * k + j] = sees ? fmaf(p, x[j], o[d][4 * k + j]) : o[d][4 * k + j];
                }
        }
}

// Output dims e .. e + 3 of a row of a sequence's block.
__device__ __forceinline__ uint64_t out_at(const AttnArgs &a, uint32_t begin, uint32_t kvh, uint32_t row) {
    const uint32_t tok = div_fast(row, a.group_div);
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

// ---- the line of tiles ------------------------------------------------------
// Every block of ROWS rows of every sequence that the launch serves, with the
// tiles of TOKENS tokens that its rows may see, once per key/value head: head
// after head, in each sequence after sequence, block after block, tile after tile.
// Workgroups take equal parts of the line, so that the load is even whatever the
// lengths are, and blocks next to each other, which read the same keys, run on one
// XCD at about the same time. A block begins with START places without a tile, for what
// it costs besides its tiles (its rows, its pages, the first loads, its results).

// Which sequences a launch serves: those of `least` to `most` rows (new tokens *
// group) per key/value head.
struct RowRange {
    uint32_t least, most;
};

// A sequence's first token row, its rows' tokens and its length.
struct Seq {
    uint32_t begin, n;
    int32_t len;
};
// The batch's start and len: copies in LDS where there are few sequences (one fetch for
// the whole workgroup, where every later look would wait for a cache, a microsecond at
// the kernel's start), else themselves. Pointers that may be either, so that there is one
// code for both: what a workgroup does once waits for its instructions to be fetched.
struct Seqs {
    const int32_t *start, *len;
    __device__ __forceinline__ Seq at(const AttnArgs &a, uint32_t s) const {
        Seq q;
        uint32_t end;
        seq_rows(start, a.kv.n_tokens, s, &q.begin, &end);
        q.n = end - q.begin;
        // (kept where sums with a few 2^24 do not overflow)
        q.len = min(len[s], int32_t(kMaxPos) - 64);
        return q;
    }
    __device__ __forceinline__ Seq uniform(const AttnArgs &a, uint32_t s) const {
        const Seq q = at(a, s);
        return Seq{uint32_t(__builtin_amdgcn_readfirstlane(q.begin)), uint32_t(__builtin_amdgcn_readfirstlane(q.n)),
                   __builtin_amdgcn_readfirstlane(q.len)};
    }
};
__device__ __forceinline__ uint32_t rows_in(const AttnArgs &a, RowRange rg, uint32_t n) {
    const uint32_t rows = n * a.group;
    return rows >= rg.least && rows <= rg.most ? rows : 0;
}

// A block of rows of a sequence: its positions, and its tiles.
struct RowBlock {
    uint32_t begin, rows;  // first token row; rows of the sequence (tokens * group)
    int32_t pos0;          // position of the sequence's first token
    int32_t first, last;   // positions of the block's first and last row
    int32_t lo, hi;        // tokens that a row of it may see
    uint32_t tiles;        // at least 1, so that rows which see nothing are written too
};
template <int ROWS, int TOKENS>
__device__ __forceinline__ RowBlock row_block(const AttnArgs &a, const Seq &q, uint32_t r0) {
    RowBlock b;
    b.begin = q.begin;
    b.rows = q.n * a.group;
    b.pos0 = max(q.len, 0) - int32_t(q.n);
    b.first = b.pos0 + int32_t(div_fast(r0, a.group_div));
    b.last = b.pos0 + int32_t(div_fast(min(r0 + ROWS, max(b.rows, 1u)) - 1, a.group_div));
    b.hi = max(0, min(b.last + 1, a.cap));
    b.lo = min(b.hi, max(0, max(b.first, -1) + 1 - a.span)) & ~31;
    b.tiles = max(1u, uint32_t(b.hi - b.lo + TOKENS - 1) / TOKENS);
    return b;
}

// A place on the line.
struct Place {
    uint32_t seq, r0, kvh, off;  // off: places of the block that lie before it
};

// The stretch of a block that a part with `left` places takes from place `off` on.
struct Segment {
    uint32_t places, off, tiles;  // of them, the first tile and the tiles
};
template <int START>
__device__ __forceinline__ Segment segment(uint32_t tiles, uint32_t off, uint64_t left) {
    Segment g;
    g.places = uint32_t(min(uint64_t(tiles + START - off), left));
    const uint32_t end = off + g.places;
    g.off = off > START ? off - START : 0;
    g.tiles = (end > START ? end - START : 0) - g.off;
    return g;
}

template <int THREADS>
struct LineMisc {
    int32_t start[THREADS + 1], len[THREADS];  // of up to THREADS sequences
    uint64_t blocks[THREADS];  // blocks of the sequences up to a thread's last: of few rows, of many << 32
    uint64_t waves[3][THREADS / 64];
    Place at;
};

template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t other_lane(uint64_t v) {  // 0 where there is none
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, int(uint32_t(v)), CTRL, ROWS, 15, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, int(uint32_t(v >> 32)), CTRL, ROWS, 15, false);
    return uint64_t(hi) << 32 | lo;
}
// Inclusive sum over the workgroup's threads, and the sum of all. All threads call it.
template <int THREADS>
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t (&waves)[THREADS / 64], uint32_t tid, uint64_t *all) {
    const uint32_t lane = tid & 63, wave = tid >> 6;
    v += other_lane<0x111, 15>(v);  // 1, 2, 4, 8 lanes to the left in rows of 16
    v += other_lane<0x112, 15>(v);
    v += other_lane<0x114, 15>(v);
    v += other_lane<0x118, 15>(v);
    v += other_lane<0x142, 10>(v);  // the last lane of rows 0 and 2 to rows 1 and 3
    v += other_lane<0x143, 12>(v);  // lane 31 to rows 2 and 3
    if (lane == 63) waves[wave] = v;
    __syncthreads();
    static_assert(THREADS == 512, "");
    uint64_t x = waves[lane % 8];
    x += other_lane<0x111, 15>(x);
    x += other_lane<0x112, 15>(x);
    x += other_lane<0x114, 15>(x);  // (lanes 0 to 7: the waves up to this one)
    auto upto = [&](uint32_t w) {
        return uint64_t(uint32_t(__builtin_amdgcn_readlane(uint32_t(x >> 32), w))) << 32 | uint32_t(__builtin_amdgcn_readlane(uint32_t(x), w));
    };
    *all = upto(7);
    return wave == 0 ? v : v + upto(__builtin_amdgcn_readfirstlane(wave - 1) & 7);
}

// x / y for x up to 2^53 (the compiler's division of 64-bit integers is 150 instructions,
// and what a workgroup does once waits for its instructions to be fetched)
__device__ __forceinline__ uint64_t div_wide(uint64_t x, uint64_t y) {
    if (__builtin_expect((x | y) >> 32 == 0, 1)) return uint32_t(x) / uint32_t(y);
    uint64_t q = uint64_t(double(x) / double(y));
    const int64_t r = int64_t(x - q * y);
    if (r < 0)
        --q;
    else if (uint64_t(r) >= y)
        ++q;
    return q;
}

// A line as one thread sees it: its blocks' places, and where they lie.
struct Line {
    uint32_t s, r0;      // its first block
    uint64_t places, incl;  // its places; with those of the threads before it
    uint64_t per_head;   // all of one head
};
template <int ROWS>
__device__ __forceinline__ void line_step(const AttnArgs &a, RowRange rg, Seqs seqs, uint32_t &s, uint32_t &r0) {  // to the next block
    r0 += ROWS;
    if (r0 >= rows_in(a, rg, seqs.at(a, s).n)) {
        r0 = 0;
        do ++s;
        while (s + 1 < a.kv.n_seq && rows_in(a, rg, seqs.at(a, s).n) == 0);
        s = min(s, a.kv.n_seq - 1);  // (start and len may change under a call that should not run then)
    }
}
// The sequences into LDS where they fit, and their blocks of both kinds counted: few |
// many << 32.
template <int FEW, int MANY, int THREADS>
__device__ __forceinline__ uint64_t count_blocks(const AttnArgs &a, RowRange few, RowRange many, LineMisc<THREADS> &lm, Seqs &seqs, uint32_t tid) {
    const uint32_t per = (a.kv.n_seq + THREADS - 1) / THREADS;
    seqs = Seqs{a.kv.start, a.kv.len};
    uint64_t mine = 0, all;
    for (uint32_t i = 0, s = tid * per; i < per && s < a.kv.n_seq; ++i, ++s) {
        const int32_t x = seqs.start[s], y = seqs.start[s + 1], z = seqs.len[s];
        if (per == 1) lm.start[s] = x, lm.start[s + 1] = y, lm.len[s] = z;  // (two lanes write the same)
        const int32_t se[2] = {x, y};
        uint32_t begin, end;
        seq_rows(se, a.kv.n_tokens, 0, &begin, &end);
        mine += (rows_in(a, few, end - begin) + FEW - 1) / FEW + (uint64_t((rows_in(a, many, end - begin) + MANY - 1) / MANY) << 32);
    }
    lm.blocks[tid] = block_scan<THREADS>(mine, lm.waves[0], tid, &all);
    if (per == 1) seqs = Seqs{lm.start, lm.len};
    __syncthreads();
    return all;
}
// The line of the blocks of one kind, `n_blocks` of them, whose counts stand at bit `shift`.
template <int ROWS, int TOKENS, int START, int THREADS>
__device__ __forceinline__ Line line_scan(const AttnArgs &a, RowRange rg, LineMisc<THREADS> &lm, Seqs seqs, uint32_t n_blocks, uint32_t shift, uint32_t tid) {
    const uint32_t per = (a.kv.n_seq + THREADS - 1) / THREADS;
    Line ln{0, 0, 0, 0, 0};
    // the places of this thread's blocks
    const uint32_t q = (n_blocks + THREADS - 1) / THREADS;
    const uint32_t f0 = min(tid * q, n_blocks), f1 = min(f0 + q, n_blocks);
    if (f0 < f1) {
        // the first thread whose sequences reach past block f0
        uint32_t x = 0, y = min(a.kv.n_seq, uint32_t(THREADS)) - 1;
        while (x < y) {
            const uint32_t mid = (x + y) / 2;
            if (uint32_t(lm.blocks[mid] >> shift) > f0)
                y = mid;
            else
                x = mid + 1;
        }
        uint32_t skip = f0 - (x != 0 ? uint32_t(lm.blocks[x - 1] >> shift) : 0);
        for (ln.s = x * per; ln.s + 1 < a.kv.n_seq; ++ln.s) {
            const uint32_t nb = (rows_in(a, rg, seqs.at(a, ln.s).n) + ROWS - 1) / ROWS;
            if (skip < nb) break;
            skip -= nb;
        }
        ln.r0 = skip * ROWS;
        uint32_t u = ln.s, v = ln.r0;
        for (uint32_t f = f0; f < f1; ++f) {
            ln.places += row_block<ROWS, TOKENS>(a, seqs.at(a, u), v).tiles + START;
            if (f + 1 < f1) line_step<ROWS>(a, rg, seqs, u, v);
        }
    }
    ln.incl = block_scan<THREADS>(ln.places, lm.waves[shift == 0 ? 1 : 2], tid, &ln.per_head);
    return ln;
}

// Part `index` of `parts` (of at least min_part places each): where it starts, and its
// number of places (0: none); *part: that of every part but the last ones.
template <int ROWS, int TOKENS, int START, int THREADS>
__device__ __forceinline__ Place line_part(const AttnArgs &a, RowRange rg, const Line &ln, uint32_t index, uint32_t parts,
                                           uint32_t min_part, LineMisc<THREADS> &lm, Seqs seqs, uint64_t *part, uint64_t *left) {
    const uint64_t total = ln.per_head * a.kv.kv_heads;
    *part = max(div_wide(total + parts - 1, parts), uint64_t(min_part));
    const uint64_t at = *part * index;
    *left = at < total ? min(*part, total - at) : 0;
    if (*left != 0) {
        const uint32_t kvh = min(uint32_t(div_wide(at, ln.per_head)), a.kv.kv_heads - 1);
        uint64_t target = at - kvh * ln.per_head;
        if (target >= ln.incl - ln.places && target < ln.incl) {
            target -= ln.incl - ln.places;
            uint32_t s = ln.s, r0 = ln.r0;
            for (;;) {
                const uint32_t t = row_block<ROWS, TOKENS>(a, seqs.at(a, s), r0).tiles + START;
                if (target < t) break;
                target -= t;
                line_step<ROWS>(a, rg, seqs, s, r0);
            }
            lm.at = Place{s, r0, kvh, uint32_t(target)};
        }
    }
    __syncthreads();
    Place p;
    p.seq = __builtin_amdgcn_readfirstlane(lm.at.seq);
    p.r0 = __builtin_amdgcn_readfirstlane(lm.at.r0);
    p.kvh = __builtin_amdgcn_readfirstlane(lm.at.kvh);
    p.off = __builtin_amdgcn_readfirstlane(lm.at.off);
    return p;
}

// The block of rows behind place p's (p.off = 0); false where the line ends there, as it
// only does if start or len have changed since.
template <int ROWS>
__device__ __forceinline__ bool next_block(const AttnArgs &a, RowRange rg, Seqs seqs, uint32_t rows, Place &p) {
    p.off = 0;
    p.r0 += ROWS;
    if (p.r0 < rows) return true;
    p.r0 = 0;
    do {
        if (++p.seq == a.kv.n_seq) {
            p.seq = 0;
            if (++p.kvh == a.kv.kv_heads) return false;
        }
    } while (rows_in(a, rg, seqs.uniform(a, p.seq).n) == 0);
    return true;
}

// ---- pages --------------------------------------------------------------------
// The cache rows of a stretch of tiles in LDS: for each run of 16 tokens, which lies
// in one page, its first cache row / 16, looked up by all threads at once (tile by
// tile, the chain of scalar loads took two thirds of the prompt kernel's step), and
// whether a page holds it: where none does, run 0 takes its place in the loads.
template <int STRETCH>
struct RunMisc {
    uint32_t run[2 * STRETCH];
    uint64_t held[STRETCH / 32];  // bit i % 64 of word i / 64: run i
};
// For the tiles from position pos on (a multiple of 16), whose tokens up to position
// `last` may be seen (those behind count as held).
template <int THREADS, int STRETCH>
__device__ __forceinline__ void find_runs(const AttnArgs &a, uint32_t seq, uint32_t kvh, int32_t pos, int32_t last, uint32_t tiles,
                                          RunMisc<STRETCH> &rm, uint32_t tid) {
    const uint32_t per = a.kv.page / 16;
    for (uint32_t i = tid; i / 64 * 64 < 2 * tiles; i += THREADS) {  // (whole waves)
        const int32_t p = pos + 16 * int32_t(i);
        const uint32_t pi = div_fast(uint32_t(p), a.kv.page_div);
        const bool wanted = i < 2 * tiles && p <= last;
        const int32_t pg = wanted ? page_at(a.kv, seq, pi) : -1;
        rm.run[i] = pg < 0 ? 0 : (uint32_t(pg) * a.kv.kv_heads + kvh) * per + (uint32_t(p) / 16 - pi * per);
        const uint64_t held = __ballot(pg >= 0 || !wanted);
        if (i % 64 == 0) rm.held[i / 64] = held;
    }
}
// Whether all runs of the stretch are held (a barrier after find_runs).
template <int STRETCH>
__device__ __forceinline__ bool all_held(const RunMisc<STRETCH> &rm, uint32_t tiles, uint32_t lane) {
    return __ballot(lane < (2 * tiles + 63) / 64 && rm.held[lane % (STRETCH / 32)] != ~uint64_t(0)) == 0;
}
// The two runs of a tile, wave-uniform. (Not an array: one that lanes index goes to
// memory, and waiting for that waits for every tile on its way.)
struct TileRuns {
    uint32_t first, second;
    __device__ __forceinline__ uint32_t of(bool later) const {
        const uint32_t x = first, y = second;
        return later ? y : x;
    }
};
template <int STRETCH>
__device__ __forceinline__ TileRuns tile_runs(const RunMisc<STRETCH> &rm, uint32_t t) {
    return TileRuns{uint32_t(__builtin_amdgcn_readfirstlane(rm.run[2 * t])), uint32_t(__builtin_amdgcn_readfirstlane(rm.run[2 * t + 1]))};
}
// Which of them pages hold: bit g for run g.
template <int STRETCH>
__device__ __forceinline__ uint32_t tile_held(const RunMisc<STRETCH> &rm, uint32_t t) {
    return uint32_t(rm.held[t / 32] >> (2 * (t % 32))) & 3;
}

// ---- rows of q --------------------------------------------------------------
// The lane's row, in NP pieces of the operands' type, and its factor log2(e) * scale *
// 2^e. `row` is query head row % group of the sequence's token row / group; rows at
// n_rows or above are zeros.
template <int CT, int NP>
constexpr bool f32_rows() { return NP == (CT == kBF16 ? 3 : 2); }
// its elements as they are, on their way
template <int CT, int NP, int R, int DP, int ES>
__device__ __forceinline__ void fetch_q(const AttnArgs &a, uint32_t begin, uint32_t kvh, uint32_t row, uint32_t n_rows, uint32_t g,
                                        u32x4 (&raw)[f32_rows<CT, NP>() ? 2 : 1][Geo<R, DP>::KS]) {
    constexpr int W = f32_rows<CT, NP>() ? 2 : 1;
    const uint32_t tok = div_fast(row, a.group_div);
    const uint64_t at = uint64_t(begin + tok) * a.q_stride + uint64_t(kvh * a.group + row - tok * a.group) * a.kv.dim;
#pragma unroll
    for (int ks = 0; ks < Geo<R, DP>::KS; ++ks) {
        const uint32_t d = step_dim<R, ES>(ks, g);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            raw[w][ks] = u32x4{0, 0, 0, 0};
            if (row < n_rows && d < a.kv.dim)
                raw[w][ks] = *reinterpret_cast<const u32x4 *>(static_cast<const uint8_t *>(a.q) + (at + d) * (2 * W) + 16 * w);
        }
    }
}
template <int CT, int NP, int R, int DP>
__device__ __forceinline__ float make_q(const AttnArgs &a, const u32x4 (&raw)[f32_rows<CT, NP>() ? 2 : 1][Geo<R, DP>::KS],
                                        u32x4 (&q)[NP][Geo<R, DP>::KS]) {
    constexpr int KS = Geo<R, DP>::KS;
    float x[KS][8], m = 0.0f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (f32_rows<CT, NP>()) {
                x[ks][i] = __builtin_bit_cast(float, uint32_t(raw[i / 4][ks][i % 4]));
            } else {
                const uint32_t h = i % 2 ? raw[0][ks][i / 2] >> 16 : raw[0][ks][i / 2] & 0xFFFF;
                x[ks][i] = a.xtype == kBF16 ? __builtin_bit_cast(float, h << 16) : float(__builtin_bit_cast(_Float16, uint16_t(h)));
            }
        }
    int e = 0;
    if constexpr (CT != kBF16) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(x[ks][i]));
        e = row_exponent<CT>(groups_max<R>(m));
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        if constexpr (CT != kBF16)
#pragma unroll
            for (int i = 0; i < 8; ++i) x[ks][i] = ldexpf(x[ks][i], -e);
#pragma unroll
        for (int p = 0; p < NP; ++p)
#pragma unroll
            for (int i = 0; i < 4; ++i) q[p][ks][i] = piece2<CT>(x[ks][2 * i], x[ks][2 * i + 1]);
    }
    // (not 0: times an unseen score, -inf, it stays that)
    return fmaxf(ldexpf(1.4426950408889634f * a.scale, e), 0x1p-126f);
}

// ---- the kernel's shape ---------------------------------------------------------
// 8 waves, one workgroup per CU; the small things first in LDS.
constexpr int kWaves = 8, kThreads = 64 * kWaves, kMisc = 16384, kLds = 160 * 1024;
struct Misc {
    LineMisc<kThreads> line;
    RunMisc<512> runs;
    union {
        struct {
            float m[kWaves][16], l[kWaves][16], inv[16];
        } few;
        struct {
            float kf[4][32], lv[4][32], iv[4][32];  // factors of a tile's keys; log2 and reciprocal of the values'
        } many;
    };
};
static_assert(sizeof(Misc) <= kMisc, "");

// What a workgroup has to do: a part of a line.
struct Part {
    Place at;
    uint64_t part, left;
    uint32_t id;  // of all parts
};

// ---- the join ----------------------------------------------------------------
// Blocks of rows split over several parts: the rows of the block that part x has on the
// list. Where many parts share a block a workgroup takes a row and its waves the
// parts; where few do, DP / 4 lanes take a row.
template <int DP, int SLOT>
__global__ __launch_bounds__(kThreads) void k_attn_join(AttnArgs a, SplitScratch sc) {
    const SplitJob job = sc.jobs[blockIdx.x];
    if (job.count == 0) return;
    __shared__ f32x4 part_x[kWaves][64];
    __shared__ float part_l[kWaves];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, rows = job.rows;
    constexpr uint32_t L = DP / 4;  // lanes of a row
    const uint32_t e = 4 * (tid % L);
    auto at_slot = [&](uint32_t i, uint32_t r) { return (i == 0 ? job.slot : 2 * (blockIdx.x + i)) * SLOT + r; };
    auto add = [&](uint32_t i, uint32_t r, float top, f32x4 &x, float &all) __attribute__((always_inline)) {
        const uint32_t at = at_slot(i, r);
        const float m = sc.ml[at * 2], l = sc.ml[at * 2 + 1];
        const float w = m == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(m - top);  // (no tokens: zeros)
        all = fmaf(w, l, all);
        const f32x4 p = *reinterpret_cast<const f32x4 *>(sc.o + uint64_t(at) * DP + e);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = fmaf(w, p[k], x[k]);
    };
    auto store = [&](uint32_t r, f32x4 x, float all) __attribute__((always_inline)) {
        const float inv = all == 0.0f ? 0.0f : 1.0f / all;
        if (e < a.kv.dim) store4(a, job.begin, job.kvh, job.r0 + r, e, x * inv);
    };
    if (job.count <= 8) {
        for (uint32_t r = blockIdx.y * (kThreads / L) + tid / L; r < rows; r += gridDim.y * (kThreads / L)) {
            float top = kNegInf, all = 0.0f;
            for (uint32_t i = 0; i < job.count; ++i) top = fmaxf(top, sc.ml[at_slot(i, r) * 2]);
            f32x4 x = {0, 0, 0, 0};
#pragma unroll 4
            for (uint32_t i = 0; i < job.count; ++i) add(i, r, top, x, all);
            store(r, x, all);
        }
        return;
    }
    // (64 / L parts at a time in a wave)
    constexpr uint32_t P = 64 / L;
    for (uint32_t r = blockIdx.y; r < rows; r += gridDim.y) {
        float top = kNegInf;
        for (uint32_t i = lane; i < job.count; i += 64) top = fmaxf(top, sc.ml[at_slot(i, r) * 2]);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
        f32x4 x = {0, 0, 0, 0};
        float all = 0.0f;
#pragma unroll 4
        for (uint32_t i = wave * P + lane / L; i < job.count; i += kWaves * P) add(i, r, top, x, all);
#pragma unroll
        for (uint32_t o = L; o < 64; o <<= 1) {
            all += __shfl_xor(all, int(o));
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] += __shfl_xor(x[k], int(o));
        }
        __syncthreads();
        part_x[wave][lane] = x;
        if (lane == 0) part_l[wave] = all;
        __syncthreads();
        if (tid < L) {
            for (int w = 1; w < kWaves; ++w) {
                all += part_l[w];
                x += part_x[w][lane];
            }
            store(r, x, all);
        }
    }
}

}  // namespace
}  // namespace tc
