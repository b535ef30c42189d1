// tc_attn_inst.hip -- the attention kernels for one cache type (TC_ATTN_CACHE, one
// object each), and the choice of the number of pieces and the padded head size.
#include "tc_attn_split.hpp"
#include "tc_attn_tile.hpp"

#ifndef TC_ATTN_CACHE
#define TC_ATTN_CACHE 30
#endif

namespace tc {
namespace {

template <int CT, int NP, int DP>
hipError_t split(const AttnArgs &a, RowRange rg, int num_cu, void *scratch, hipStream_t st) {
    using Sh = SplitShape<CT, NP, DP>;
    static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(&k_attn_split<CT, NP, DP>),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, Sh::LDS);
    if (attr != hipSuccess) return attr;
    const uint32_t grid = Sh::OCC * num_cu;
    const SplitScratch sc = split_scratch(scratch, grid, Sh::R);
    k_attn_split<CT, NP, DP><<<grid, 64 * Sh::NW, Sh::LDS, st>>>(a, rg, sc);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    k_attn_join<DP, Sh::R><<<dim3(grid, Sh::R / 4), 256, 0, st>>>(a, sc);
    return hipGetLastError();
}

template <int CT, int NP, int DP>
hipError_t tile(const AttnArgs &a, RowRange rg, int num_cu, void *scratch, hipStream_t st) {
    using Sh = TileShape<CT, NP, DP>;
    static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(&k_attn_tile<CT, NP, DP>),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, Sh::LDS);
    if (attr != hipSuccess) return attr;
    const uint32_t grid = Sh::OCC * num_cu;
    const SplitScratch sc = split_scratch(scratch, grid, Sh::ROWS);
    k_attn_tile<CT, NP, DP><<<grid, 64 * Sh::NW, Sh::LDS, st>>>(a, rg, sc);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    k_attn_join<DP, Sh::ROWS><<<dim3(grid, Sh::ROWS / 4), 256, 0, st>>>(a, sc);
    return hipGetLastError();
}

// Sequences of few rows and of many go to different kernels. The lengths are the
// device's, so both are launched unless the call's size rules one out; a kernel
// without work ends at once.
template <int CT, int NP, int DP>
hipError_t both(const AttnArgs &a, int num_cu, void *scratch, hipStream_t st) {
    const uint64_t most = uint64_t(a.kv.n_tokens) * a.group;
    if (a.kv.n_seq > 1 || most <= kSplitRows) {
        const hipError_t e = split<CT, NP, DP>(a, RowRange{1, kSplitRows}, num_cu, scratch, st);
        if (e != hipSuccess || most <= kSplitRows) return e;
    }
    return tile<CT, NP, DP>(a, RowRange{a.kv.n_seq > 1 ? kSplitRows + 1 : 1, ~0u}, num_cu, scratch, st);
}

template <int CT, int NP>
hipError_t by_dim(const AttnArgs &a, int num_cu, void *scratch, hipStream_t st) {
    if (a.kv.dim <= 64) return both<CT, NP, 64>(a, num_cu, scratch, st);
    if (a.kv.dim <= 128) return both<CT, NP, 128>(a, num_cu, scratch, st);
    return both<CT, NP, 256>(a, num_cu, scratch, st);
}

}  // namespace

// Pieces of q and of the weights: what a row's type has bits for.
template <>
hipError_t launch_attn_cache<TC_ATTN_CACHE>(const AttnArgs &a, int num_cu, void *scratch, hipStream_t st) {
    constexpr int CT = TC_ATTN_CACHE;
    if constexpr (CT == kBF16) {
        if (a.xtype == kF32) return by_dim<CT, 3>(a, num_cu, scratch, st);
        if (a.xtype == kF16) return by_dim<CT, 2>(a, num_cu, scratch, st);
    } else {
        if (a.xtype == kF32) return by_dim<CT, 2>(a, num_cu, scratch, st);
    }
    return by_dim<CT, 1>(a, num_cu, scratch, st);
}

}  // namespace tc
