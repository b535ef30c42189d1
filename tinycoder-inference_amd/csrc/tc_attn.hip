// tc_attn.hip -- causal attention of a chunk of new tokens over a paged cache.
#include "tc_attn_common.hpp"
#include "tc_kernels.hpp"

namespace tc {
namespace {

constexpr uint32_t kTile = 64;

template <int CT>
__device__ __forceinline__ float cache_at(const uint8_t *c, uint64_t i) {
    if constexpr (CT == kF16) return h2f(reinterpret_cast<const uint16_t *>(c)[i]);
    if constexpr (CT == kBF16) return __builtin_bit_cast(float, uint32_t(reinterpret_cast<const uint16_t *>(c)[i]) << 16);
    if constexpr (CT == kI8) return float(int8_t(c[i]));
    return __builtin_amdgcn_cvt_f32_fp8(int(c[i]), 0);
}

// One wave per (row, query head): a lane per token for the scores, lanes over
// the dims for the weighted sum, running maximum and sum.
template <int CT>
__global__ __launch_bounds__(64) void k_attn_rows(AttnArgs a) {
    __shared__ float qs[kMaxHeadDim], ps[kTile];
    __shared__ int64_t rows[kTile];
    const uint32_t h = blockIdx.x, kvh = h / a.group, lane = threadIdx.x, D = a.kv.dim;
    for (uint32_t s = blockIdx.z; s < a.kv.n_seq; s += gridDim.z) {
        uint32_t b, e;
        seq_rows(a.kv.start, a.kv.n_tokens, s, &b, &e);
        const int64_t len = a.kv.len[s];
        for (uint32_t t = b + blockIdx.y; t < e; t += gridDim.y) {
            const int64_t pos = len - (e - t);
            const uint64_t qo = uint64_t(t) * a.q_stride + h * D;
            __syncthreads();
            for (uint32_t i = lane; i < D; i += 64) {
                float x;
                if (a.xtype == kF32) x = static_cast<const float *>(a.q)[qo + i];
                else if (a.xtype == kF16) x = h2f(static_cast<const uint16_t *>(a.q)[qo + i]);
                else x = __builtin_bit_cast(float, uint32_t(static_cast<const uint16_t *>(a.q)[qo + i]) << 16);
                qs[i] = x;
            }
            const int64_t lo = a.window && pos >= a.window ? pos - a.window + 1 : 0;
            float m = -__builtin_inff(), l = 0.0f, acc[4] = {0, 0, 0, 0};
            for (int64_t j0 = lo; j0 <= pos; j0 += kTile) {
                const int64_t j = j0 + lane;
                const int64_t row = j <= pos ? cache_row(a.kv, s, j, kvh) : -1;
                float x = -__builtin_inff();
                __syncthreads();
                rows[lane] = row;
                if (row >= 0) {
                    float d = 0.0f;
                    for (uint32_t i = 0; i < D; ++i) d = fmaf(qs[i], cache_at<CT>(a.kv.k, uint64_t(row) * D + i), d);
                    if constexpr (scaled_type(CT)) d *= a.kv.ks[row];
                    x = d * a.scale;
                }
                float mx = x;
                for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
                const float mn = fmaxf(m, mx);
                const float ref = mn == -__builtin_inff() ? 0.0f : mn;
                const float al = __expf(m - ref);
                const float p = row >= 0 ? __expf(x - ref) : 0.0f;
                float sum = p;
                for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
                l = l * al + sum;
                m = mn;
                ps[lane] = row >= 0 && scaled_type(CT) ? p * a.kv.vs[row] : p;
                __syncthreads();
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t i = lane + 64 * k;
                    if (i >= D) break;
                    float v = acc[k] * al;
                    for (uint32_t c = 0; c < kTile; ++c)
                        if (rows[c] >= 0) v = fmaf(ps[c], cache_at<CT>(a.kv.v, uint64_t(rows[c]) * D + i), v);
                    acc[k] = v;
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t i = lane + 64 * k;
                if (i >= D) break;
                const float o = l > 0.0f || l != l ? acc[k] / l : 0.0f;
                const uint64_t at = (uint64_t(t) * a.heads + h) * D + i;
                if (a.xtype == kF32) static_cast<float *>(a.out)[at] = o;
                else if (a.xtype == kF16) static_cast<_Float16 *>(a.out)[at] = _Float16(o);
                else static_cast<__bf16 *>(a.out)[at] = __bf16(o);
            }
        }
    }
}

}  // namespace

size_t attn_scratch_bytes(uint32_t, uint32_t, int) { return 0; }

hipError_t launch_attn(const AttnArgs &a, int ctype, int, void *, hipStream_t st) {
    const uint32_t zs = a.kv.n_seq < 1024 ? a.kv.n_seq : 1024;
    const uint32_t per = (a.kv.n_tokens + a.kv.n_seq - 1) / a.kv.n_seq;
    const dim3 grid(a.heads, per < 1024 ? per : 1024, zs);
    switch (ctype) {
        case kF16: k_attn_rows<kF16><<<grid, 64, 0, st>>>(a); break;
        case kBF16: k_attn_rows<kBF16><<<grid, 64, 0, st>>>(a); break;
        case kI8: k_attn_rows<kI8><<<grid, 64, 0, st>>>(a); break;
        default: k_attn_rows<kE4M3><<<grid, 64, 0, st>>>(a); break;
    }
    return hipGetLastError();
}

}  // namespace tc
