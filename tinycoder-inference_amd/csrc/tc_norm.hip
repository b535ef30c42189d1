// tc_norm.hip -- residual stream, gate and norms between two blocks, in one pass.
//
//   h' = h + scale * gate * post(y),   x = pre(h'),   norm(z) = (z - mean) / sqrt(mean(z^2) + eps) * w + b
//
// A workgroup has a row (a wave of it, where rows are short), held in registers from its load
// to its stores: y and h are read once, h' and x written once, and the statistics of both
// norms, of a layer norm's differences too, come from the registers in fp32: a sum over a
// lane's values, over the wave, over the waves through LDS. So the kernel is bound by HBM for
// many rows, and for few by the chain of one load, one sum over the row per statistic, and the
// store; the weights' loads are issued in front of the sums.
#include "tc_actquant.hpp"
#include "tc_kernels.hpp"
#include "tc_step.hpp"

namespace tc {
namespace {

__device__ __forceinline__ float load1(int type, const void *p, uint64_t elem) {
    if (type == kF32) return static_cast<const float *>(p)[elem];
    const uint32_t w = static_cast<const uint16_t *>(p)[elem];
    return type == kF16 ? h2f(w) : __builtin_bit_cast(float, w << 16);
}
__device__ __forceinline__ void store1(int type, void *p, uint64_t elem, float x) {
    if (type == kF32)
        static_cast<float *>(p)[elem] = x;
    else
        static_cast<uint16_t *>(p)[elem] = uint16_t(type == kF16 ? pack_f16(x, 0.0f) : pack_bf16(x, 0.0f));
}

// A lane's 8 values of a row from column `at` on, zeros behind the row's end. VEC: all 8
// inside the row or none, and 16-byte aligned; else its columns are `at` + 64 i.
template <bool VEC>
__device__ __forceinline__ void row_load(int type, const void *p, uint64_t row, uint32_t at, uint32_t cols, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.0f;
    if constexpr (VEC) {
        if (at < cols) load8(type, p, row + at, x);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (at + 64 * i < cols) x[i] = load1(type, p, row + at + 64 * i);
    }
}
template <bool VEC>
__device__ __forceinline__ void row_store(int type, void *p, uint64_t row, uint32_t at, uint32_t cols, const float (&x)[8]) {
    if constexpr (VEC) {
        if (at < cols) store8(type, p, row + at, x);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (at + 64 * i < cols) store1(type, p, row + at + 64 * i, x[i]);
    }
}

__device__ __forceinline__ float wave_sum(float v) {
    v += dpp_f<0x111>(v);  // 1, 2, 4, 8 lanes to the left in rows of 16: lane 15 of each has its sum
    v += dpp_f<0x112>(v);
    v += dpp_f<0x114>(v);
    v += dpp_f<0x118>(v);
    const int b = __builtin_bit_cast(int, v);
    auto lane = [&](int l) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, l)); };
    return (lane(15) + lane(31)) + (lane(47) + lane(63));
}

// Sum over the row's lanes; `at` counts the sums of a row, so that two barriers are not needed
// for each: every one has its own place.
template <bool ONE>
__device__ __forceinline__ float row_sum(float v, float *lds, int at) {
    v = wave_sum(v);
    if constexpr (ONE) return v;
    const uint32_t waves = blockDim.x >> 6, lane = threadIdx.x & 63;
    if (lane == 0) lds[16 * at + (threadIdx.x >> 6)] = v;
    __syncthreads();
    return wave_sum(lane < waves ? lds[16 * at + lane] : 0.0f);
}

// One row normed in place; first: the number of its first sum.
template <bool VEC, bool ONE, int C>
__device__ __forceinline__ void norm_row(const NormArgs &n, uint32_t cols, uint32_t at, uint32_t step, float *lds, int first,
                                         float (&z)[C][8]) {
    // (long rows have no registers for them so early)
    constexpr bool EARLY = C <= 2;
    float w[C][8], b[C][8];
    auto load = [&](int c) {
        if (n.weight != nullptr) row_load<VEC>(kF32, n.weight, 0, at + c * step, cols, w[c]);
        if (n.bias != nullptr) row_load<VEC>(kF32, n.bias, 0, at + c * step, cols, b[c]);
    };
    if constexpr (EARLY)
#pragma unroll
        for (int c = 0; c < C; ++c) load(c);
    const float inv_n = 1.0f / float(cols);
    if (n.kind == TC_NORM_LAYER) {
        float s = 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) s += z[c][i];
        const float mean = row_sum<ONE>(s, lds, first) * inv_n;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                z[c][i] = at + c * step + (VEC ? 0 : 64 * i) < cols ? z[c][i] - mean : 0.0f;
    }
    // (squares times a power of two near 1 / cols, so that their sum passes fp32's range no sooner
    // than the largest square does)
    const float down = __builtin_bit_cast(float, (127u - (32u - __builtin_clz(cols))) << 23);
    float s = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) s = __builtin_fmaf(z[c][i] * down, z[c][i], s);
    const float inv = rsqrtf(__builtin_fmaf(row_sum<ONE>(s, lds, first + 1), inv_n / down, n.eps));
#pragma unroll
    for (int c = 0; c < C; ++c) {
        if constexpr (!EARLY) load(c);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            z[c][i] *= inv;
            if (n.weight != nullptr) z[c][i] *= w[c][i] + n.offset;
            if (n.bias != nullptr) z[c][i] += b[c][i];
        }
    }
}

__device__ __forceinline__ float sigmoid(float g) { return 1.0f / (1.0f + expf(-g)); }

// C: blocks of 8 values of a lane. ONE: a wave has a row, a workgroup four; else a
// workgroup has one. ACT: quantized activations too.
template <bool VEC, bool ONE, int C, bool ACT>
__global__ __launch_bounds__(ONE ? 256 : 1024) void k_norm(NormCall a) {
    __shared__ float lds[64];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t r = ONE ? blockIdx.x * 4 + wave : blockIdx.x;
    if (r >= a.rows) return;  // (only where no barrier follows)
    const uint32_t w0 = ONE ? 0 : wave, waves = ONE ? 1 : blockDim.x >> 6;
    // a lane's blocks lie a row of lanes apart
    const uint32_t at = w0 * 512 + (VEC ? lane * 8 : lane), step = waves * 512, cols = a.cols;
    float h[C][8];
    if (a.y != nullptr) {
        float y[C][8], g[C][8];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            row_load<VEC>(a.y_type, a.y, r * a.y_stride, at + c * step, cols, y[c]);
            row_load<VEC>(a.h_type, a.h, r * a.h_stride, at + c * step, cols, h[c]);
        }
        float row_gate = a.scale;
        if (a.gate_kind == TC_GATE_ROW) {
            const float v = load1(a.gate_type, a.gate, r);
            row_gate *= a.gate_sigmoid ? sigmoid(v) : v;
        } else if (a.gate_kind != TC_GATE_NONE) {
            const uint64_t base = a.gate_kind == TC_GATE_FULL ? uint64_t(r) * cols : 0;
#pragma unroll
            for (int c = 0; c < C; ++c) row_load<VEC>(a.gate_type, a.gate, base, at + c * step, cols, g[c]);
        }
        if (a.post.kind >= 0) norm_row<VEC, ONE, C>(a.post, cols, at, step, lds, 0, y);
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float f = row_gate;
                if (a.gate_kind == TC_GATE_CHANNEL || a.gate_kind == TC_GATE_FULL)
                    f *= a.gate_sigmoid ? sigmoid(g[c][i]) : g[c][i];
                h[c][i] = __builtin_fmaf(f, y[c][i], h[c][i]);
            }
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (a.h_out != nullptr) row_store<VEC>(a.h_type, a.h_out, r * a.h_out_stride, at + c * step, cols, h[c]);
            // (a bias of `post` is not to count behind the row's end)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (at + c * step + (VEC ? 0 : 64 * i) >= cols) h[c][i] = 0.0f;
        }
    } else {
#pragma unroll
        for (int c = 0; c < C; ++c) row_load<VEC>(a.h_type, a.h, r * a.h_stride, at + c * step, cols, h[c]);
    }
    if (a.pre.kind < 0) return;
    norm_row<VEC, ONE, C>(a.pre, cols, at, step, lds, 2, h);
    if (a.x != nullptr)
#pragma unroll
        for (int c = 0; c < C; ++c) row_store<VEC>(a.x_type, a.x, r * a.x_stride, at + c * step, cols, h[c]);
    if constexpr (ACT) {
        // the quantizers want a block of 256 columns in a wave, four to a lane
        extern __shared__ float row[];
#pragma unroll
        for (int c = 0; c < C; ++c)
            if (at + c * step < cols) {
                f32x4 *p = reinterpret_cast<f32x4 *>(row + at + c * step);
                p[0] = f32x4{h[c][0], h[c][1], h[c][2], h[c][3]};
                p[1] = f32x4{h[c][4], h[c][5], h[c][6], h[c][7]};
            }
        __syncthreads();
        const uint32_t blocks = cols >> 8;
        for (uint32_t b = wave; b < blocks; b += waves) {
            const float4 v = reinterpret_cast<const float4 *>(row + b * 256)[lane];
            const size_t o = size_t(r) * blocks + b;
            if (a.act_q8_0)
                quant_q8_0_blocks_wave_v(v, a.qs + o * 256, a.d + o * 8, a.dg + o * 32);
            else
                quant_q8k_block_wave_v(v, a.qs + o * 256, a.d + o, a.bsums + o * 16, a.dg + o * 16);
        }
    }
}

template <bool VEC, bool ONE, int C>
hipError_t launch(const NormCall &a, uint32_t waves, hipStream_t st) {
    if (a.qs != nullptr) {
        if constexpr (VEC && !ONE && C <= 2)
            k_norm<VEC, ONE, C, true><<<a.rows, 64 * waves, a.cols * 4, st>>>(a);
        else
            return hipErrorInvalidValue;  // (not reached: launch_norm)
    } else if (ONE) {
        k_norm<VEC, ONE, C, false><<<(a.rows + 3) / 4, 256, 0, st>>>(a);
    } else {
        k_norm<VEC, ONE, C, false><<<a.rows, 64 * waves, 0, st>>>(a);
    }
    return hipGetLastError();
}

template <bool VEC>
hipError_t launch(const NormCall &a, int num_cu, hipStream_t st) {
    const uint32_t blocks = (a.cols + 511) / 512;  // of a wave's 512 columns
    if (blocks == 1 && a.qs == nullptr) return launch<VEC, true, 1>(a, 1, st);
    const bool many = a.rows > 4u * uint32_t(num_cu);
    const uint32_t c = blocks > 32 ? 4 : blocks > 16 || (many && blocks > 1) ? 2 : 1;
    const uint32_t waves = (blocks + c - 1) / c;
    switch (c) {
        case 1: return launch<VEC, false, 1>(a, waves, st);
        case 2: return launch<VEC, false, 2>(a, waves, st);
        default: return launch<VEC, false, 4>(a, waves, st);
    }
}

}  // namespace

hipError_t launch_norm(const NormCall &a, int num_cu, hipStream_t st) {
    // rows that 16-byte accesses cut into whole parts
    auto fits = [&](const void *p, uint64_t stride, int type) {
        return p == nullptr || ((reinterpret_cast<uintptr_t>(p) & 15) == 0 && (a.rows == 1 || stride * elem_bytes(type) % 16 == 0));
    };
    const bool gate = a.gate_kind == TC_GATE_CHANNEL || a.gate_kind == TC_GATE_FULL;
    const bool vec = a.cols % 8 == 0 && fits(a.h, a.h_stride, a.h_type) && fits(a.y, a.y_stride, a.y_type) &&
                     fits(a.h_out, a.h_out_stride, a.h_type) && fits(a.x, a.x_stride, a.x_type) &&
                     (!gate || fits(a.gate, a.gate_kind == TC_GATE_FULL ? a.cols : 0, a.gate_type)) && fits(a.post.weight, 0, kF32) &&
                     fits(a.post.bias, 0, kF32) && fits(a.pre.weight, 0, kF32) && fits(a.pre.bias, 0, kF32);
    return vec ? launch<true>(a, num_cu, st) : launch<false>(a, num_cu, st);
}

}  // namespace tc
