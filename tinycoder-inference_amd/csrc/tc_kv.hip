// tc_kv.hip -- keys and values into a paged cache, quantized on the way, and
// back out of it.
//
// A row of one head (dim values) is the unit: a group of lanes, 8 values each,
// loads it, agrees on its largest magnitude (8-bit types), and stores it with
// one 16- or 8-byte store per lane. Nothing is read twice, so both kernels are
// bound by HBM for long chunks and by the chain batch -> page table -> store for
// short ones; the rows' loads are issued before that chain, and long chunks give a
// lane four rows, whose chains run side by side. Up to 16 tokens of a head are next to
// each other: they are in the cache, where one token's heads lie a page apart.
//
// The 8-bit types hold one factor per row: scores and the weights of the values
// then take it as one product per token, after the matrix cores, where factors
// for parts of a row would have to go into the operands.
#include "tc_attn_common.hpp"
#include "tc_kernels.hpp"

namespace tc {
namespace {

constexpr uint32_t kThreads = 256;

// Largest of `lanes` lanes' values (a power of two; no NaN) in each of them.
__device__ __forceinline__ float group_max(float v, uint32_t lanes) {
    for (uint32_t o = 1; o < lanes; o <<= 1) v = fmaxf(v, __shfl_xor(v, int(o)));
    return v;
}

// How a launch goes over the rows: a block of 2^tokens token rows after the other, in it
// the keys of head after head, then the values, a token after the other.
struct Walk {
    uint32_t rows;     // of a workgroup at a time
    uint32_t lanes;    // of a row
    DivMod lane_div;   // by lanes
    DivMod block_div;  // by a block's rows
    uint32_t tokens;   // log2 of a block's tokens
};
struct Row {
    uint32_t t, h;  // token row, head
    bool second;    // value (not key)
    bool live;      // a row of the call, and values of it the lane's
};
template <int U>
struct Rows {
    Row r[U];
    uint32_t i;  // first of the lane's 8 values
    int seq;     // of the first of the workgroup's tokens
};

// The lane's rows, and the sequence of the first token among the workgroup's.
template <int U>
__device__ __forceinline__ Rows<U> rows_of(const KvArgs &a, const Walk &w) {
    Rows<U> p;
    const uint32_t mine = div_fast(threadIdx.x, w.lane_div), base = blockIdx.x * U * w.rows;
    p.i = (threadIdx.x - mine * w.lanes) * 8;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t r = base + u * w.rows + mine, b = div_fast(r, w.block_div), in = r - b * w.block_div.d;
        const uint32_t j = in >> w.tokens;
        p.r[u].t = (b << w.tokens) + (in & ((1u << w.tokens) - 1));
        p.r[u].second = j >= a.kv_heads;
        p.r[u].h = p.r[u].second ? j - a.kv_heads : j;
        p.r[u].live = mine < w.rows && p.r[u].t < a.n_tokens && p.i < a.dim;
    }
    const uint32_t first = min(div_fast(base, w.block_div) << w.tokens, a.n_tokens - 1);
    p.seq = wave_find_seq(a.start, a.n_seq, first);
    return p;
}
// Sequences and cache rows of the lane's rows (-1: none).
template <int U>
__device__ __forceinline__ void find_slots(const KvArgs &a, const Rows<U> &p, int (&seq)[U], int64_t (&row)[U]) {
    const int32_t end = p.seq >= 0 ? a.start[p.seq + 1] : 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        seq[u] = p.seq;
        if (int32_t(p.r[u].t) >= end) seq[u] = find_seq(a.start, a.n_seq, min(p.r[u].t, a.n_tokens - 1));
    }
#pragma unroll
    for (int u = 0; u < U; ++u) row[u] = slot_of(a, seq[u], p.r[u].t, p.r[u].h);
}

// One row to where it belongs.
template <int CT>
__device__ __forceinline__ void put(const KvArgs &a, const Row &r, uint32_t at, int64_t row, uint32_t lanes, const float (&x)[8]) {
    uint8_t *dst = r.second ? a.v : a.k;
    if constexpr (!scaled_type(CT)) {
        if (r.live && row >= 0) store8(CT, dst, uint64_t(row) * a.dim + at, x);
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
        if (!r.live || row < 0) return;
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
        *reinterpret_cast<u32x2 *>(dst + uint64_t(row) * a.dim + at) = u32x2{w[0], w[1]};
        if (at == 0) (r.second ? a.vs : a.ks)[row] = d;
    }
}

template <int CT, int U>
__global__ __launch_bounds__(kThreads) void k_kv_write(KvArgs a, int xtype, const void *k, const void *v, uint32_t k_stride,
                                                       uint32_t v_stride, Walk w) {
    const Rows<U> p = rows_of<U>(a, w);
    float x[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const Row &r = p.r[u];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[u][i] = 0.0f;
        if (r.live) load8(xtype, r.second ? v : k, uint64_t(r.t) * (r.second ? v_stride : k_stride) + r.h * a.dim + p.i, x[u]);
    }
    int seq[U];
    int64_t row[U];
    find_slots<U>(a, p, seq, row);
#pragma unroll
    for (int u = 0; u < U; ++u) put<CT>(a, p.r[u], p.i, row[u], w.lanes, x[u]);
}

template <int CT, int U>
__global__ __launch_bounds__(kThreads) void k_kv_read(KvArgs a, int xtype, void *k, void *v, Walk w) {
    const Rows<U> p = rows_of<U>(a, w);
    int seq[U];
    int64_t row[U];
    find_slots<U>(a, p, seq, row);
    float x[U][8], d[U];
    u32x2 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint8_t *src = p.r[u].second ? a.v : a.k;
        const bool there = p.r[u].live && row[u] >= 0;
        if constexpr (scaled_type(CT)) {
            raw[u] = u32x2{0, 0}, d[u] = 0.0f;
            if (there) {
                raw[u] = *reinterpret_cast<const u32x2 *>(src + uint64_t(row[u]) * a.dim + p.i);
                d[u] = (p.r[u].second ? a.vs : a.ks)[row[u]];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[u][i] = 0.0f;
            if (there) load8(CT, src, uint64_t(row[u]) * a.dim + p.i, x[u]);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if constexpr (scaled_type(CT))
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t q = raw[u][i];
                if constexpr (CT == kI8) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[u][4 * i + j] = float(int8_t(q >> (8 * j))) * d[u];
                } else {
                    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(int(q), false);
                    const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(int(q), true);
                    x[u][4 * i] = lo[0] * d[u], x[u][4 * i + 1] = lo[1] * d[u];
                    x[u][4 * i + 2] = hi[0] * d[u], x[u][4 * i + 3] = hi[1] * d[u];
                }
            }
        // (rows past the last sequence stay as they are)
        if (p.r[u].live && seq[u] >= 0)
            store8(xtype, p.r[u].second ? v : k, (uint64_t(p.r[u].t) * a.kv_heads + p.r[u].h) * a.dim + p.i, x[u]);
    }
}

// `group`: a row's lanes agree on something, so they are a power of two.
Walk make_walk(const KvArgs &a, bool group, uint32_t *passes) {
    Walk w;
    w.lanes = a.dim / 8;
    if (group)
        for (w.lanes = 2; w.lanes * 8 < a.dim;) w.lanes *= 2;
    w.rows = kThreads / w.lanes;
    w.tokens = 0;
    while (w.tokens < 4 && (2u << w.tokens) <= a.n_tokens) ++w.tokens;
    const uint32_t block = (2 * a.kv_heads) << w.tokens, blocks = (a.n_tokens + (1u << w.tokens) - 1) >> w.tokens;
    w.lane_div = make_divmod(w.lanes);
    w.block_div = make_divmod(block);
    *passes = (blocks * block + w.rows - 1) / w.rows;
    return w;
}

// Four rows of a lane from where single ones are more than the card holds at a time: 177 MB
// read out 61 -> 43 us (two 45, eight 46), while 18 MB written take 10.4 us so and 12.8
// with four, 13 MB read 5.3 and 6.8.
constexpr uint32_t kPasses = 4096;

template <int CT>
hipError_t write(const KvArgs &a, int xtype, const void *k, const void *v, uint32_t k_stride, uint32_t v_stride, hipStream_t st) {
    uint32_t passes;
    const Walk w = make_walk(a, scaled_type(CT), &passes);
    if (passes < kPasses)
        k_kv_write<CT, 1><<<passes, kThreads, 0, st>>>(a, xtype, k, v, k_stride, v_stride, w);
    else
        k_kv_write<CT, 4><<<(passes + 3) / 4, kThreads, 0, st>>>(a, xtype, k, v, k_stride, v_stride, w);
    return hipGetLastError();
}

template <int CT>
hipError_t read(const KvArgs &a, int xtype, void *k, void *v, hipStream_t st) {
    uint32_t passes;
    const Walk w = make_walk(a, false, &passes);
    if (passes < kPasses)
        k_kv_read<CT, 1><<<passes, kThreads, 0, st>>>(a, xtype, k, v, w);
    else
        k_kv_read<CT, 4><<<(passes + 3) / 4, kThreads, 0, st>>>(a, xtype, k, v, w);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_kv_write(const KvArgs &a, int ctype, int xtype, const void *k, const void *v, uint32_t k_stride,
                           uint32_t v_stride, hipStream_t st) {
    switch (ctype) {
        case kF16: return write<kF16>(a, xtype, k, v, k_stride, v_stride, st);
        case kBF16: return write<kBF16>(a, xtype, k, v, k_stride, v_stride, st);
        case kI8: return write<kI8>(a, xtype, k, v, k_stride, v_stride, st);
        default: return write<kE4M3>(a, xtype, k, v, k_stride, v_stride, st);
    }
}

hipError_t launch_kv_read(const KvArgs &a, int ctype, int xtype, void *k, void *v, hipStream_t st) {
    switch (ctype) {
        case kF16: return read<kF16>(a, xtype, k, v, st);
        case kBF16: return read<kBF16>(a, xtype, k, v, st);
        case kI8: return read<kI8>(a, xtype, k, v, st);
        default: return read<kE4M3>(a, xtype, k, v, st);
    }
}

}  // namespace tc
