// tc_kv.hip -- keys and values into a paged cache, quantized on the way, and
// back out of it.
//
// A row of one head (dim values) is the unit: a group of lanes, 8 values each,
// loads it, agrees on its largest magnitude (8-bit types), and stores it with
// one 16- or 8-byte store per lane. Nothing is read twice, so both kernels are
// bound by HBM for long chunks and by the chain batch -> page table -> store for
// short ones; the rows' loads are issued before that chain.
//
// The 8-bit types hold one factor per row: scores and the weights of the values
// then take it as one product per token, after the matrix cores, where factors
// for parts of a row would have to go into the operands.
#include "tc_attn_common.hpp"
#include "tc_kernels.hpp"

namespace tc {
namespace {

constexpr uint32_t kThreads = 256;

// Largest of `lpr` lanes' values (a power of two; no NaN) in each of them.
__device__ __forceinline__ float group_max(float v, uint32_t lpr) {
    for (uint32_t o = 1; o < lpr; o <<= 1) v = fmaxf(v, __shfl_xor(v, int(o)));
    return v;
}

// A lane's part in a launch over 2 * n_tokens * kv_heads rows, keys and values
// of a token next to each other.
struct Part {
    uint32_t t, h, i;  // token row, head, first of the lane's 8 values
    bool second, live, has;  // value (not key); a row of the call; values in it
};
__device__ __forceinline__ Part part(const KvArgs &a, uint32_t lpr, DivMod per_token) {
    const uint64_t r = (uint64_t(blockIdx.x) * kThreads + threadIdx.x) / lpr;
    Part p;
    p.live = r < uint64_t(a.n_tokens) * 2 * a.kv_heads;
    const uint32_t r32 = p.live ? uint32_t(r) : 0;
    p.t = div_fast(r32, per_token);
    const uint32_t w = r32 - p.t * 2 * a.kv_heads;
    p.second = w >= a.kv_heads;
    p.h = p.second ? w - a.kv_heads : w;
    p.i = threadIdx.x % lpr * 8;
    p.has = p.live && p.i < a.dim;
    return p;
}

template <int CT>
__global__ __launch_bounds__(kThreads) void k_kv_write(KvArgs a, int xtype, const void *k, const void *v, uint32_t k_stride,
                                                       uint32_t v_stride, uint32_t lpr, DivMod per_token) {
    const Part p = part(a, lpr, per_token);
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (p.has) load8(xtype, p.second ? v : k, uint64_t(p.t) * (p.second ? v_stride : k_stride) + p.h * a.dim + p.i, x);
    const int64_t row = p.live ? slot_of(a, find_seq(a.start, a.n_seq, p.t), p.t, p.h) : -1;
    uint8_t *dst = p.second ? a.v : a.k;
    if constexpr (!scaled_type(CT)) {
        if (p.has && row >= 0) store8(CT, dst, uint64_t(row) * a.dim + p.i, x);
    } else {
        float m = 0.0f;
        bool odd = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            m = fmaxf(m, fabsf(x[i]));
            odd = odd || x[i] != x[i];
        }
        // a NaN makes the factor infinite, as an infinity does: the row reads
        // back as 0 * inf
        m = group_max(odd ? __builtin_inff() : m, lpr);
        constexpr float top = CT == kI8 ? 127.0f : 448.0f;
        float d = __fdiv_rn(m, top);
        if (d == 0.0f) d = 1.0f;  // zeros, and what is so small that the factor would be
        if (!p.has || row < 0) return;
        uint32_t w[2];
        if constexpr (CT == kI8) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                w[i] = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float q = __builtin_rintf(__fdiv_rn(x[4 * i + j], d));
                    // (a quotient over an infinite factor may be NaN: 0)
                    const int n = q == q ? int(fminf(fmaxf(q, -127.0f), 127.0f)) : 0;
                    w[i] |= (uint32_t(n) & 0xFF) << (8 * j);
                }
            }
        } else {
            float q[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                q[i] = __fdiv_rn(x[i], d);
                q[i] = q[i] == q[i] ? fminf(fmaxf(q[i], -448.0f), 448.0f) : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                int u = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i], q[4 * i + 1], 0, false);
                w[i] = uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i + 2], q[4 * i + 3], u, true));
            }
        }
        *reinterpret_cast<u32x2 *>(dst + uint64_t(row) * a.dim + p.i) = u32x2{w[0], w[1]};
        if (p.i == 0) (p.second ? a.vs : a.ks)[row] = d;
    }
}

template <int CT>
__global__ __launch_bounds__(kThreads) void k_kv_read(KvArgs a, int xtype, void *k, void *v, uint32_t lpr, DivMod per_token) {
    const Part p = part(a, lpr, per_token);
    if (!p.has) return;
    const int s = find_seq(a.start, a.n_seq, p.t);
    if (s < 0) return;  // rows past the last sequence stay as they are
    const int64_t row = slot_of(a, s, p.t, p.h);
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (row >= 0) {
        const uint8_t *src = p.second ? a.v : a.k;
        if constexpr (!scaled_type(CT)) {
            load8(CT, src, uint64_t(row) * a.dim + p.i, x);
        } else {
            const u32x2 w = *reinterpret_cast<const u32x2 *>(src + uint64_t(row) * a.dim + p.i);
            const float d = (p.second ? a.vs : a.ks)[row];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t u = w[i];
                if constexpr (CT == kI8) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[4 * i + j] = float(int8_t(u >> (8 * j))) * d;
                } else {
                    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(int(u), false);
                    const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(int(u), true);
                    x[4 * i] = lo[0] * d, x[4 * i + 1] = lo[1] * d, x[4 * i + 2] = hi[0] * d, x[4 * i + 3] = hi[1] * d;
                }
            }
        }
    }
    store8(xtype, p.second ? v : k, (uint64_t(p.t) * a.kv_heads + p.h) * a.dim + p.i, x);
}

// Lanes per row and workgroups of a launch.
uint32_t shape(const KvArgs &a, uint32_t *lpr) {
    *lpr = 2;
    while (*lpr * 8 < a.dim) *lpr *= 2;
    return uint32_t((uint64_t(a.n_tokens) * 2 * a.kv_heads * *lpr + kThreads - 1) / kThreads);
}

}  // namespace

hipError_t launch_kv_write(const KvArgs &a, int ctype, int xtype, const void *k, const void *v, uint32_t k_stride,
                           uint32_t v_stride, hipStream_t st) {
    uint32_t lpr;
    const uint32_t grid = shape(a, &lpr);
    const DivMod pt = make_divmod(2 * a.kv_heads);
    switch (ctype) {
        case kF16: k_kv_write<kF16><<<grid, kThreads, 0, st>>>(a, xtype, k, v, k_stride, v_stride, lpr, pt); break;
        case kBF16: k_kv_write<kBF16><<<grid, kThreads, 0, st>>>(a, xtype, k, v, k_stride, v_stride, lpr, pt); break;
        case kI8: k_kv_write<kI8><<<grid, kThreads, 0, st>>>(a, xtype, k, v, k_stride, v_stride, lpr, pt); break;
        default: k_kv_write<kE4M3><<<grid, kThreads, 0, st>>>(a, xtype, k, v, k_stride, v_stride, lpr, pt); break;
    }
    return hipGetLastError();
}

hipError_t launch_kv_read(const KvArgs &a, int ctype, int xtype, void *k, void *v, hipStream_t st) {
    uint32_t lpr;
    const uint32_t grid = shape(a, &lpr);
    const DivMod pt = make_divmod(2 * a.kv_heads);
    switch (ctype) {
        case kF16: k_kv_read<kF16><<<grid, kThreads, 0, st>>>(a, xtype, k, v, lpr, pt); break;
        case kBF16: k_kv_read<kBF16><<<grid, kThreads, 0, st>>>(a, xtype, k, v, lpr, pt); break;
        case kI8: k_kv_read<kI8><<<grid, kThreads, 0, st>>>(a, xtype, k, v, lpr, pt); break;
        default: k_kv_read<kE4M3><<<grid, kThreads, 0, st>>>(a, xtype, k, v, lpr, pt); break;
    }
    return hipGetLastError();
}

}  // namespace tc
