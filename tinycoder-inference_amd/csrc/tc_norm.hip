// tc_norm.hip -- residual stream, gate and norms between two blocks, in one pass.
//
//   h' = h + scale * gate * post(y),   x = pre(h'),   norm(z) = (z - mean) / sqrt(mean(z^2) + eps) * w + b
//
// A row is held in registers from its load to its stores, by a workgroup or, where it is short,
// by 8 to 64 lanes: y and h are read once, h' and x written once, and the statistics of both norms,
// of a layer norm's differences too, come from the registers in fp32: a sum over a lane's values,
// over the wave, over the waves through LDS. So many rows are bound by HBM (8192 rows of 5120, bf16,
// with both norms: 67 us, 336 MB at 5.0 TB/s, a large copy's rate; VALU 0.37 busy), and few by the
// chain of one load, one sum over the row per statistic, the weights and the store (one row of
// 3584 2.8 us, of which a launch is 2.4).
//
// Not kept: workgroups that go through many rows with the weights in registers and the next row on
// its way (8192 rows 112 us: fewer rows of a CU at work), stores past the caches (67 -> 64, but
// 2 more with the next kernel's reads).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "tc_actquant.hpp"
#include "tc_kernels.hpp"
#include "tc_step.hpp"

namespace tc {
namespace {

__device__ __forceinline__ void store1(int type, void *p, uint64_t elem, float x) {
    if (type == kF32)
        static_cast<float *>(p)[elem] = x;
    else
        static_cast<uint16_t *>(p)[elem] = uint16_t(type == kF16 ? pack_f16(x, 0.0f) : pack_bf16(x, 0.0f));
}

// 16 bytes at any address that fits their elements (rows of odd widths and strides): the
// hardware takes such accesses whole.
typedef uint32_t u32x4d __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4h __attribute__((ext_vector_type(4), aligned(2)));

// A lane's 8 columns of a row: from `at` on. The lane at the row's end has the row's last 8,
// of which the first `off` are the lane's before it; lanes behind it have off = 8. (So every lane
// loads 16 bytes, and no branch parts the loads: with one for each type and end, a load waited
// for the one before it.)
struct Span {
    uint32_t at, off;
};

// A lane's 8 values as they are in memory (16-bit types: a alone).
struct Raw {
    u32x4 a, b;
};
// W: the elements' bytes. TINY: rows of less than 8 columns, all of them the first lane's.
template <int W, bool TINY>
__device__ __forceinline__ Raw raw_load(const void *p, uint64_t row, Span s, uint32_t cols) {
    Raw r;
    if constexpr (TINY) {
        r.a = r.b = u32x4{0, 0, 0, 0};
        if (s.off < 8)
#pragma unroll
            for (int i = 0; i < 7; ++i)
                if (uint32_t(i) < cols) {
                    if constexpr (W == 4)
                        (i < 4 ? r.a : r.b)[i & 3] = static_cast<const uint32_t *>(p)[row + i];
                    else
                        r.a[i >> 1] |= uint32_t(static_cast<const uint16_t *>(p)[row + i]) << (16 * (i & 1));
                }
    } else if constexpr (W == 4) {
        const u32x4d *q = reinterpret_cast<const u32x4d *>(static_cast<const float *>(p) + row + s.at);
        r.a = q[0], r.b = q[1];
    } else {
        r.a = *reinterpret_cast<const u32x4h *>(static_cast<const uint16_t *>(p) + row + s.at);
    }
    return r;
}
template <int W>
__device__ __forceinline__ void widen(int type, const Raw &r, float (&x)[8]) {
    if constexpr (W == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __builtin_bit_cast(float, uint32_t(r.a[i])), x[4 + i] = __builtin_bit_cast(float, uint32_t(r.b[i]));
    } else if (type == kF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[2 * i] = h2f(r.a[i] & 0xFFFF), x[2 * i + 1] = h2f(r.a[i] >> 16);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __builtin_bit_cast(float, uint32_t(r.a[i]) << 16);
            x[2 * i + 1] = __builtin_bit_cast(float, r.a[i] & 0xFFFF0000u);
        }
    }
}
// Zeros in the place of what is not the lane's own.
template <bool TINY>
__device__ __forceinline__ void own_only(Span s, uint32_t cols, float (&x)[8]) {
    if (s.off == 0 && !TINY) return;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (TINY ? s.off == 8 || uint32_t(i) >= cols : uint32_t(i) < s.off) x[i] = 0.0f;
}
template <int W, bool TINY>
__device__ __forceinline__ void row_store(int type, void *p, uint64_t row, Span s, uint32_t cols, const float (&x)[8]) {
    if (s.off == 0 && !TINY) {
        if constexpr (W == 4) {
            u32x4d *q = reinterpret_cast<u32x4d *>(static_cast<float *>(p) + row + s.at);
            q[0] = __builtin_bit_cast(u32x4, f32x4{x[0], x[1], x[2], x[3]});
            q[1] = __builtin_bit_cast(u32x4, f32x4{x[4], x[5], x[6], x[7]});
        } else {
            u32x4 u;
#pragma unroll
            for (int i = 0; i < 4; ++i) u[i] = type == kF16 ? pack_f16(x[2 * i], x[2 * i + 1]) : pack_bf16(x[2 * i], x[2 * i + 1]);
            *reinterpret_cast<u32x4h *>(static_cast<uint16_t *>(p) + row + s.at) = u;
        }
    } else if (s.off != 8) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (TINY ? uint32_t(i) < cols : uint32_t(i) >= s.off) store1(type, p, row + s.at + i, x[i]);
    }
}
template <bool TINY>
__device__ __forceinline__ void row_store(int type, void *p, uint64_t row, Span s, uint32_t cols, const float (&x)[8]) {
    type == kF32 ? row_store<4, TINY>(type, p, row, s, cols, x) : row_store<2, TINY>(type, p, row, s, cols, x);
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

// Sum over the row's lanes: LANES of a wave (a power of two), or a workgroup's (0). Every sum of a
// row has its own place in LDS, so that one barrier is enough for each.
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float *lds) {
    if constexpr (LANES == 64) {
        return wave_sum(v);
    } else if constexpr (LANES != 0) {
        v += dpp_f<0xB1>(v);  // 1, 2, 4, 8 lanes away (as quads, quads' halves and rows mirrored)
        v += dpp_f<0x4E>(v);
        v += dpp_f<0x141>(v);
        if constexpr (LANES >= 16) v += dpp_f<0x140>(v);
        if constexpr (LANES >= 32) v += __shfl_xor(v, 16);
        return v;
    } else {
        v = wave_sum(v);
        const uint32_t waves = blockDim.x >> 6, lane = threadIdx.x & 63;
        if (lane == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        return wave_sum(lane < waves ? lds[lane] : 0.0f);
    }
}

// One row normed in place; lds: places of two sums. (The weights are loaded behind the sums: held
// in registers across them they took more of a CU's rows than their way from L2 costs.)
template <int LANES, int C, bool TINY>
__device__ __forceinline__ void norm_row(const NormCall &a, const NormArgs &n, const Span (&at)[C], float *lds, float (&z)[C][8]) {
    const uint32_t cols = a.cols;
    if (n.kind == TC_NORM_LAYER) {
        float s = 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) s += z[c][i];
        const float mean = row_sum<LANES>(s, lds) * a.inv_cols;
#pragma unroll
        for (int c = 0; c < C; ++c) {
#pragma unroll
            for (int i = 0; i < 8; ++i) z[c][i] -= mean;
            own_only<TINY>(at[c], cols, z[c]);
        }
    }
    // (squares times a power of two, 1 / cols or just below, so that their sum passes fp32's range no
    // sooner than the largest square does)
    float s = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) s = __builtin_fmaf(z[c][i] * a.down, z[c][i], s);
    const float inv = rsqrtf(__builtin_fmaf(row_sum<LANES>(s, lds + 16), a.inv_cols_down, n.eps));
    Raw w[C];
    if (n.weight != nullptr)
#pragma unroll
        for (int c = 0; c < C; ++c) w[c] = raw_load<4, TINY>(n.weight, 0, at[c], cols);
#pragma unroll
    for (int c = 0; c < C; ++c) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) z[c][i] *= inv;
        if (n.weight != nullptr) {
            widen<4>(kF32, w[c], v);
#pragma unroll
            for (int i = 0; i < 8; ++i) z[c][i] *= v[i] + n.offset;
        }
        if (n.bias != nullptr) {
            widen<4>(kF32, raw_load<4, TINY>(n.bias, 0, at[c], cols), v);
#pragma unroll
            for (int i = 0; i < 8; ++i) z[c][i] += v[i];
        }
    }
}

__device__ __forceinline__ float sigmoid(float g) { return __builtin_amdgcn_rcpf(1.0f + expf(-g)); }

// YW, HW: bytes of y's (0: none) and h's elements. POST: there may be a norm of y. LANES: lanes
// that have a row, 0: the workgroup. C: blocks of 8 values of a lane. ACT: quantized activations
// too. MOST: threads of a workgroup at most (fewer leave more registers to each).
template <int YW, int HW, bool POST, int LANES, int C, bool ACT, int MOST, bool TINY>
__global__ __launch_bounds__(MOST) void k_norm(NormCall a) {
    __shared__ float lds[64];
    const uint32_t tid = threadIdx.x, lane = LANES ? tid % (LANES ? LANES : 1) : tid & 63, wave = LANES ? 0 : tid >> 6;
    const uint32_t waves = LANES ? 1 : blockDim.x >> 6, cols = a.cols;
    const uint32_t r = LANES ? blockIdx.x * (MOST / (LANES ? LANES : 1)) + tid / (LANES ? LANES : 1) : blockIdx.x;
    if (r >= a.rows) return;  // (only where no barrier follows; a row's lanes go together)
    Span at[C];  // a lane's blocks lie a row of lanes apart
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const uint32_t from = (c * waves + wave) * 512 + lane * 8;
        at[c].at = TINY ? 0 : min(from, cols - 8);
        at[c].off = TINY ? (lane ? 8 : 0) : min(from - at[c].at, 8u);
    }
    // What a block needs of h, of the gate and (where no norm comes first) of y. Long rows have two
    // blocks' on their way at a time, so that a CU has room for two rows (17407 columns 61 -> 56
    // us), others all of them.
    constexpr bool WHOLE = C <= 2;
    constexpr int SLOTS = WHOLE ? C : 2;
    Raw y_raw[POST ? C : SLOTS], h_raw[SLOTS], g_raw[SLOTS];
    const bool gated = YW != 0 && (a.gate_kind == TC_GATE_CHANNEL || a.gate_kind == TC_GATE_FULL);
    const uint64_t gate_row = a.gate_kind == TC_GATE_FULL ? uint64_t(r) * cols : 0;
    auto fetch = [&](int c) {
        if constexpr (YW != 0 && !POST) y_raw[c % SLOTS] = raw_load<YW, TINY>(a.y, r * a.y_stride, at[c], cols);
        h_raw[c % SLOTS] = raw_load<HW, TINY>(a.h, r * a.h_stride, at[c], cols);
        if (gated)
            g_raw[c % SLOTS] = a.gate_type == kF32 ? raw_load<4, TINY>(a.gate, gate_row, at[c], cols) : raw_load<2, TINY>(a.gate, gate_row, at[c], cols);
    };
    if constexpr (POST)
#pragma unroll
        for (int c = 0; c < C; ++c) y_raw[c] = raw_load<YW, TINY>(a.y, r * a.y_stride, at[c], cols);
    uint32_t row_gate = 0;
    if (YW != 0 && a.gate_kind == TC_GATE_ROW)
        row_gate = a.gate_type == kF32 ? static_cast<const uint32_t *>(a.gate)[r] : static_cast<const uint16_t *>(a.gate)[r];
#pragma unroll
    for (int c = 0; c < (WHOLE ? C : 1); ++c) fetch(c);
    float h[C][8], y[POST || WHOLE ? C : 1][8];
    if constexpr (POST) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            widen<YW>(a.y_type, y_raw[c], y[c]);
            own_only<TINY>(at[c], cols, y[c]);
        }
        if (a.post.kind >= 0) norm_row<LANES, C, TINY>(a, a.post, at, lds, y);
    }
    auto open = [&](int c) {
        widen<HW>(a.h_type, h_raw[c % SLOTS], h[c]);
        own_only<TINY>(at[c], cols, h[c]);
        if constexpr (YW != 0 && !POST) {
            float(&v)[8] = y[WHOLE ? c : 0];
            widen<YW>(a.y_type, y_raw[c % SLOTS], v);
            own_only<TINY>(at[c], cols, v);
        }
    };
    if constexpr (WHOLE)
#pragma unroll
        for (int c = 0; c < C; ++c) open(c);
    float f = a.scale;
    if (YW != 0 && a.gate_kind == TC_GATE_ROW) {
        const float v = a.gate_type == kF32   ? __builtin_bit_cast(float, row_gate)
                        : a.gate_type == kF16 ? h2f(row_gate)
                                              : __builtin_bit_cast(float, row_gate << 16);
        f *= a.gate_sigmoid ? sigmoid(v) : v;
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
        if constexpr (!WHOLE) {
            if (c + 1 < C) fetch(c + 1);
            open(c);
        }
        if constexpr (YW != 0) {
            float(&v)[8] = y[POST || WHOLE ? c : 0];
            if (gated) {
                float g[8];
                if (a.gate_type == kF32)
                    widen<4>(kF32, g_raw[c % SLOTS], g);
                else
                    widen<2>(a.gate_type, g_raw[c % SLOTS], g);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] *= a.gate_sigmoid ? sigmoid(g[i]) : g[i];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) h[c][i] = __builtin_fmaf(f, v[i], h[c][i]);
            if (a.h_out != nullptr) row_store<HW, TINY>(a.h_type, a.h_out, r * a.h_out_stride, at[c], cols, h[c]);
            own_only<TINY>(at[c], cols, h[c]);  // (`post` may have a bias, a gate infinities)
        }
        if constexpr (!WHOLE) __builtin_amdgcn_sched_barrier(0);  // (or all loads move to the front again)
    }
    if (a.pre.kind < 0) return;
    norm_row<LANES, C, TINY>(a, a.pre, at, lds + 32, h);
    if (a.x != nullptr)
#pragma unroll
        for (int c = 0; c < C; ++c) row_store<TINY>(a.x_type, a.x, r * a.x_stride, at[c], cols, h[c]);
    if constexpr (ACT) {
        // the quantizers want a block of 256 columns in a wave, four to a lane
        extern __shared__ float row[];
#pragma unroll
        for (int c = 0; c < C; ++c)
            if (at[c].off == 0) {
                f32x4 *p = reinterpret_cast<f32x4 *>(row + at[c].at);
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

// Short rows by as many lanes as they have eights (200000 rows of 128 columns 96 us with a wave
// each, 38 with 16 lanes). Others by a workgroup: one block a lane where there are few rows, whose sums
// are short then; two from 512 rows on, of which a CU holds more (16-bit rows of 5120, us with one and with two: 500 rows
// 6.35 and 6.8, 520 7.6 and 7.2, 8192 65 and 61; with a norm behind the block 6.95 and 7.2, 8.8 and 7.8, 76 and 65);
// as many as 1024 threads leave from 8192 columns on.
template <int YW, int HW, bool POST>
hipError_t launch(const NormCall &a, int num_cu, hipStream_t st) {
    const uint32_t blocks = (a.cols + 511) / 512;  // of a wave's 512 columns
    const bool many = a.rows > 2u * uint32_t(num_cu);
    auto waves = [&](uint32_t c) { return 64 * ((blocks + c - 1) / c); };
    auto grid = [&](uint32_t lanes) { return (a.rows + 256 / lanes - 1) / (256 / lanes); };
    if (a.cols <= 64)
        k_norm<YW, HW, POST, 8, 1, false, 256, false><<<grid(8), 256, 0, st>>>(a);
    else if (a.cols <= 128)
        k_norm<YW, HW, POST, 16, 1, false, 256, false><<<grid(16), 256, 0, st>>>(a);
    else if (a.cols <= 256)
        k_norm<YW, HW, POST, 32, 1, false, 256, false><<<grid(32), 256, 0, st>>>(a);
    else if (blocks == 1)
        k_norm<YW, HW, POST, 64, 1, false, 256, false><<<grid(64), 256, 0, st>>>(a);
    else if (blocks <= 16 && many)
        k_norm<YW, HW, POST, 0, 2, false, 512, false><<<a.rows, waves(2), 0, st>>>(a);
    else if (blocks <= 16)
        k_norm<YW, HW, POST, 0, 1, false, 1024, false><<<a.rows, waves(1), 0, st>>>(a);
    else if (blocks <= 32)
        k_norm<YW, HW, POST, 0, 2, false, 1024, false><<<a.rows, waves(2), 0, st>>>(a);
    else if (blocks <= 48)
        k_norm<YW, HW, POST, 0, 3, false, 1024, false><<<a.rows, waves(3), 0, st>>>(a);
    else
        k_norm<YW, HW, POST, 0, 4, false, 1024, false><<<a.rows, waves(4), 0, st>>>(a);
    return hipGetLastError();
}
template <int YW, int HW>
hipError_t launch(const NormCall &a, int num_cu, hipStream_t st) {
    const uint32_t blocks = (a.cols + 511) / 512;
    constexpr bool POST = YW != 0;
    if (a.cols < 8) {
        k_norm<YW, HW, POST, 64, 1, false, 256, true><<<(a.rows + 3) / 4, 256, 0, st>>>(a);
    } else if (a.qs != nullptr) {
        if (blocks <= 16)
            k_norm<YW, HW, POST, 0, 1, true, 1024, false><<<a.rows, 64 * blocks, a.cols * 4, st>>>(a);
        else
            k_norm<YW, HW, POST, 0, 2, true, 1024, false><<<a.rows, 64 * ((blocks + 1) / 2), a.cols * 4, st>>>(a);
    } else {
        return POST && a.post.kind >= 0 ? launch<YW, HW, POST>(a, num_cu, st) : launch<YW, HW, false>(a, num_cu, st);
    }
    return hipGetLastError();
}

hipError_t launch(const NormCall &a, int num_cu, hipStream_t st) {
    const bool wide = a.h_type == kF32;
    if (a.y == nullptr) return wide ? launch<0, 4>(a, num_cu, st) : launch<0, 2>(a, num_cu, st);
    if (a.y_type == kF32) return wide ? launch<4, 4>(a, num_cu, st) : launch<4, 2>(a, num_cu, st);
    return wide ? launch<2, 4>(a, num_cu, st) : launch<2, 2>(a, num_cu, st);
}

// `rows` rows further on.
template <class T>
T *on(T *p, uint64_t rows, uint64_t bytes) {
    using Byte = std::conditional_t<std::is_const_v<T>, const char, char>;
    return p == nullptr ? p : reinterpret_cast<T *>(reinterpret_cast<Byte *>(p) + rows * bytes);
}

constexpr uint32_t kRowsMost = 1u << 21;  // of a launch: a grid has less than 2^32 threads

}  // namespace

hipError_t launch_norm(const NormCall &call, int num_cu, hipStream_t st) {
    NormCall a = call;
    int up = 0;
    while ((1u << up) < a.cols) ++up;
    a.inv_cols = 1.0f / float(a.cols);
    a.down = std::ldexp(1.0f, -up);
    a.inv_cols_down = std::ldexp(a.inv_cols, up);
    for (uint32_t left = call.rows;;) {
        a.rows = std::min(left, kRowsMost);
        const hipError_t e = launch(a, num_cu, st);
        if (e != hipSuccess || (left -= a.rows) == 0) return e;
        const uint64_t h_bytes = elem_bytes(a.h_type), x_bytes = elem_bytes(a.x_type), block = a.act_q8_0 ? 32 : 256;
        a.h = on(a.h, a.rows, a.h_stride * h_bytes);
        a.y = on(a.y, a.rows, a.y_stride * elem_bytes(a.y_type));
        a.h_out = on(a.h_out, a.rows, a.h_out_stride * h_bytes);
        a.x = on(a.x, a.rows, a.x_stride * x_bytes);
        if (a.gate_kind == TC_GATE_ROW || a.gate_kind == TC_GATE_FULL)
            a.gate = on(a.gate, a.rows, (a.gate_kind == TC_GATE_ROW ? 1 : a.cols) * elem_bytes(a.gate_type));
        a.qs = on(a.qs, a.rows, a.cols);
        a.d = on(a.d, a.rows, a.cols / block * 4);
        a.bsums = on(a.bsums, a.rows, a.cols / 16 * 2);
        a.dg = on(a.dg, a.rows, a.cols / 256 * (a.act_q8_0 ? 32 : 16) * 2);
    }
}

}  // namespace tc
