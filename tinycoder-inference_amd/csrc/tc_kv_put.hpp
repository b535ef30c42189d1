// tc_kv_put.hpp -- a row of values into a paged cache, quantized on the way: what
// tc_kv_write and tc_rope_kv_write share.
#pragma once

#include "tc_attn_common.hpp"

namespace tc {

// op over the values of `lanes` lanes (a power of two up to 32) in each of them: 1, 2, 4 and 8
// lanes away as quads, quads' halves and rows mirrored (lane moves that go without LDS), then 16.
template <class Op>
__device__ __forceinline__ float group_all(float v, uint32_t lanes, Op op) {
    v = op(v, dpp_f<0xB1>(v));
    if (lanes > 2) v = op(v, dpp_f<0x4E>(v));
    if (lanes > 4) v = op(v, dpp_f<0x141>(v));
    if (lanes > 8) v = op(v, dpp_f<0x140>(v));
    if (lanes > 16) v = op(v, __shfl_xor(v, 16));
    return v;
}
// (no NaN)
__device__ __forceinline__ float group_max(float v, uint32_t lanes) {
    return group_all(v, lanes, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float group_sum(float v, uint32_t lanes) {
    return group_all(v, lanes, [](float a, float b) { return a + b; });
}

// The lane's 8 values x from dim `at` on of one row to cache row `row` (below 0: none) of
// dst; `lanes` lanes (a power of two) have the row between them. `live`: the lane has values
// of a row. All lanes of the row call it.
template <int CT>
__device__ __forceinline__ void put_row(uint8_t *dst, float *scales, uint32_t dim, int64_t row, uint32_t at, bool live,
                                        uint32_t lanes, const float (&x)[8]) {
    if constexpr (!scaled_type(CT)) {
        if (live && row >= 0) store8(CT, dst, uint64_t(row) * dim + at, x);
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
        m = group_max(odd ? __builtin_inff() : m, lanes);
        constexpr float top = CT == kI8 ? 127.0f : 448.0f;
        float d = __fdiv_rn(m, top);
        if (d == 0.0f) d = 1.0f;  // zeros, and what is so small that the factor would be
        if (!live || row < 0) return;
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
        *reinterpret_cast<u32x2 *>(dst + uint64_t(row) * dim + at) = u32x2{w[0], w[1]};
        if (at == 0) scales[row] = d;
    }
}

}  // namespace tc
