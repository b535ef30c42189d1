// tc_attn_inst.hip -- the attention kernels for one cache type (TC_ATTN_CACHE, one
// object each), and the choice of the number of pieces and the padded head size.
#include "tc_attn_few.hpp"
#include "tc_attn_many.hpp"

#ifndef TC_ATTN_CACHE
#define TC_ATTN_CACHE 30
#endif

namespace tc {
namespace {

// One launch for a batch of any mix: sequences of few rows make one line of tiles,
// those of many another, and the workgroups are shared out between the two as their
// tiles are (a tile of either takes about as long: 16 KB through HBM on one of 256
// CUs, or 256 rows' products): 16 sequences of drafted tokens 61 us in two launches, 35
// in one (whose few-row part also went from 4 waves to 8).
template <int CT, int NP, int DP>
__global__ __launch_bounds__(kThreads, 1) void k_attn(AttnArgs a, SplitScratch sc) {
    using Few = FewShape<CT, NP, DP>;
    using Many = ManyShape<CT, NP, DP>;
    constexpr int SLOT = Many::ROWS;
    constexpr RowRange few{1, kFewRows}, many{kFewRows + 1, ~0u};
    extern __shared__ __align__(1024) unsigned char lds[];
    Misc &ms = *reinterpret_cast<Misc *>(lds);
    const uint32_t tid = threadIdx.x, b = blockIdx.x, parts = gridDim.x;
    Seqs seqs;
    const uint64_t blocks = count_blocks<Few::R, Many::ROWS>(a, few, many, ms.line, seqs, tid);
    Line lf{}, lm{};
    if (uint32_t(blocks) != 0) lf = line_scan<Few::R, kTileTokens, Few::START>(a, few, ms.line, seqs, uint32_t(blocks), 0, tid);
    if (blocks >> 32 != 0) lm = line_scan<Many::ROWS, kTileTokens, Many::START>(a, many, ms.line, seqs, uint32_t(blocks >> 32), 32, tid);
    const uint64_t all = lf.per_head + lm.per_head;
    if (all == 0) {
        if (tid == 0) sc.jobs[b].count = 0;
        return;
    }
    uint32_t nm = lm.per_head != 0 ? parts : 0, before = lm.per_head != 0 ? b : 0;  // workgroups for the second line
    bool second = lm.per_head != 0;
    if (lf.per_head != 0 && lm.per_head != 0) {  // (spread evenly)
        nm = min(max(uint32_t(div_wide(lm.per_head * parts + all / 2, all)), 1u), parts - 1);
        before = b * nm / parts;
        second = (b + 1) * nm / parts != before;
    }
    Part w;
    if (!second) {
        const uint32_t index = b - before;
        w.at = line_part<Few::R, kTileTokens, Few::START>(a, few, lf, index, parts - nm, Few::NW, ms.line, seqs, &w.part, &w.left);
        w.id = index;
        if (tid == 0) sc.jobs[w.id].count = 0;
        attn_few<CT, NP, DP, SLOT>(a, few, seqs, sc, w, lds, ms);
    } else {
        // (workgroups of one XCD, every eighth, take parts next to each other)
        const uint32_t index = nm == parts && parts % 8 == 0 ? b % 8 * (parts / 8) + b / 8 : before;
        w.at = line_part<Many::ROWS, kTileTokens, Many::START>(a, many, lm, index, nm, 4, ms.line, seqs, &w.part, &w.left);
        w.id = parts - nm + index;
        if (tid == 0) sc.jobs[w.id].count = 0;
        attn_many<CT, NP, DP, SLOT>(a, many, seqs, sc, w, lds, ms);
    }
}

template <int CT, int NP, int DP>
hipError_t launch(const AttnArgs &a, int num_cu, void *scratch, hipStream_t st) {
    constexpr int SLOT = ManyShape<CT, NP, DP>::ROWS;
    constexpr int few = FewShape<CT, NP, DP>::LDS, many = ManyShape<CT, NP, DP>::LDS, lds = few > many ? few : many;
    static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(&k_attn<CT, NP, DP>),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (attr != hipSuccess) return attr;
    const SplitScratch sc = split_scratch(scratch, num_cu, SLOT);
    k_attn<CT, NP, DP><<<num_cu, kThreads, lds, st>>>(a, sc);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    k_attn_join<DP, SLOT><<<dim3(num_cu, 8), kThreads, 0, st>>>(a, sc);
    return hipGetLastError();
}

template <int CT, int NP>
hipError_t by_dim(const AttnArgs &a, int num_cu, void *scratch, hipStream_t st) {
    if (a.kv.dim <= 64) return launch<CT, NP, 64>(a, num_cu, scratch, st);
    if (a.kv.dim <= 128) return launch<CT, NP, 128>(a, num_cu, scratch, st);
    return launch<CT, NP, 256>(a, num_cu, scratch, st);
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
