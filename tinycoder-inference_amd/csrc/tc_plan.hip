// tc_plan.hip -- the geometry of a step from its sequences' lengths.
//
// Two sums over the sequences in their order (rows; pages wanted, given back) decide
// everything, so one workgroup forms them, 1024 sequences at a time, and enters the pages;
// with it done, a row's sequence, position and slot are looked up as the other kernels do. Few rows
// are looked up by the same workgroup: a second launch costs 4 us of a decode step's 8 to
// 10, while one workgroup's stores reach some 60 GB/s, 16 bytes a row.
//
// Sums of rows saturate at n_tokens, sums of pages at 2^30: both stay in 32 bits whatever the
// arrays hold, and min(a + b, top) is associative for numbers that are not negative.
#include "tc_kernels.hpp"
#include "tc_step.hpp"

namespace tc {
namespace {

constexpr uint32_t kThreads = 1024;
constexpr uint32_t kWaves = kThreads / 64;

struct Totals {
    uint32_t wave[kWaves];
};

// Sum of v over the threads before this one, and over all (in *all); saturating at `top`.
// Every thread calls it.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t top, Totals &lds, uint32_t *all) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t sum = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t b = uint32_t(__shfl_up(int(sum), o));
        if (lane >= uint32_t(o)) sum = min(sum + b, top);
    }
    __syncthreads();  // (the totals of the call before have been read)
    if (lane == 63) lds.wave[wave] = sum;
    __syncthreads();
    uint32_t w = lane < kWaves ? lds.wave[lane] : 0;
#pragma unroll
    for (int o = 1; o < int(kWaves); o <<= 1) {
        const uint32_t b = uint32_t(__shfl_up(int(w), o));
        if (lane >= uint32_t(o)) w = min(w + b, top);
    }
    *all = uint32_t(__shfl(int(w), kWaves - 1));
    uint32_t before = uint32_t(__shfl(int(w), int(wave) - 1 < 0 ? 0 : int(wave) - 1));
    if (wave == 0) before = 0;
    const uint32_t mine = uint32_t(__shfl_up(int(sum), 1));
    return lane == 0 ? before : min(before + mine, top);
}

__device__ __forceinline__ uint32_t bounded(int32_t v, uint32_t most) { return v < 0 ? 0u : min(uint32_t(v), most); }
// Place of the ring, `by` (up to 2^30) from place `at` on.
__device__ __forceinline__ uint32_t around(uint32_t at, uint32_t by, uint32_t ring) {
    uint32_t i = at + by;  // (ring, at and by are at most 2^30)
    if (i >= ring) i -= ring;
    return i >= ring ? i % ring : i;
}

// Sequence, position and slot of a row.
__device__ __forceinline__ void put_row_maps(const tc_plan &a, const DivMod &page, uint32_t t, int seq) {
    int32_t pos = -1;
    int64_t slot = -1;
    if (seq >= 0) {
        pos = a.len[seq] - a.start[seq + 1] + int32_t(t);
        // (a length that was held to the largest leaves its first rows no position)
        if (pos >= 0) {
            const uint32_t pi = div_fast(uint32_t(pos), page);
            if (pi < a.table_pages) {
                const int32_t pg = a.table[size_t(seq) * a.table_pages + pi];
                if (pg >= 0) slot = int64_t(pg) * a.page_tokens + (uint32_t(pos) - pi * a.page_tokens);
            }
        } else {
            pos = -1;
        }
    }
    if (a.sequence) a.sequence[t] = seq;
    if (a.position) a.position[t] = pos;
    if (a.slot) a.slot[t] = slot;
}

__global__ __launch_bounds__(kThreads) void k_plan(tc_plan a, DivMod page, uint32_t rows) {
    __shared__ Totals lds;
    const uint32_t S = a.n_seq, R = a.ring_pages, W = a.table_pages, lane = threadIdx.x & 63;
    const uint32_t at = bounded(a.free[0], R - 1), left0 = bounded(a.free[1], R);
    // pages of ended sequences behind the free ones
    uint32_t back_all = 0;
    for (uint32_t s0 = 0; s0 < S; s0 += kThreads) {
        const uint32_t s = s0 + threadIdx.x;
        const uint32_t back = s < S && a.new_tokens[s] < 0 ? bounded(a.pages[s], W) : 0;
        uint32_t all;
        const uint32_t before = min(back_all + block_scan(back, kPlanMost, lds, &all), kPlanMost);
        back_all = min(back_all + all, kPlanMost);
        // a wave takes its sequences one after the other, a lane a page
        for (uint64_t m = __ballot(back != 0); m != 0; m &= m - 1) {
            const int l = __builtin_ctzll(m);
            const uint32_t n = __builtin_amdgcn_readlane(back, l), b = __builtin_amdgcn_readlane(before, l);
            const uint32_t room = left0 + b < R ? R - left0 - b : 0;
            const int32_t *row = a.table + size_t(s0 + (threadIdx.x & ~63u) + l) * W;
            for (uint32_t j = lane; j < min(n, room); j += 64) a.ring[around(at, left0 + b + j, R)] = row[j];
        }
    }
    const uint32_t left = min(left0 + back_all, R);
    __threadfence_block();
    __syncthreads();
    uint32_t row_all = 0, want_all = 0, short_all = 0;
    for (uint32_t s0 = 0; s0 < S; s0 += kThreads) {
        const uint32_t s = s0 + threadIdx.x;
        const int32_t fresh = s < S ? a.new_tokens[s] : -1;
        const uint32_t held = s < S ? bounded(a.held[s], kLenMost) : 0, had = s < S ? bounded(a.pages[s], W) : 0;
        uint32_t all;
        const uint32_t n = bounded(fresh, a.n_tokens);
        const uint32_t begin = min(row_all + block_scan(n, a.n_tokens, lds, &all), a.n_tokens);
        row_all = min(row_all + all, a.n_tokens);
        const uint32_t got_rows = min(n, a.n_tokens - begin);
        const uint32_t len = fresh < 0 ? 0 : min(held + got_rows, uint32_t(kLenMost));
        uint32_t need = div_fast(len, page);
        if (need * a.page_tokens < len) ++need;
        const uint32_t fit = min(need, W), want = fresh >= 0 && fit > had ? fit - had : 0;
        const uint32_t before = min(want_all + block_scan(want, kPlanMost, lds, &all), kPlanMost);
        want_all = min(want_all + all, kPlanMost);
        block_scan(need - fit, kPlanMost, lds, &all);
        short_all = min(short_all + all, kPlanMost);
        // the first page by the sequence's own lane, more of them by its wave
        if (want != 0) a.table[size_t(s) * W + had] = before < left ? a.ring[around(at, before, R)] : -1;
        for (uint64_t m = __ballot(want > 1); m != 0; m &= m - 1) {
            const int l = __builtin_ctzll(m);
            const uint32_t k = __builtin_amdgcn_readlane(want, l), b = __builtin_amdgcn_readlane(before, l);
            int32_t *row = a.table + size_t(s0 + (threadIdx.x & ~63u) + l) * W + __builtin_amdgcn_readlane(had, l);
            for (uint32_t j = 1 + lane; j < k; j += 64) row[j] = b + j < left ? a.ring[around(at, b + j, R)] : -1;
        }
        if (s < S) {
            a.start[s] = int32_t(begin);
            a.len[s] = int32_t(len);
            a.pages_out[s] = fresh < 0 ? 0 : int32_t(had + (before < left ? min(want, left - before) : 0));
        }
    }
    if (threadIdx.x == 0) {
        const uint32_t taken = min(want_all, left);
        a.start[S] = int32_t(row_all);
        a.free_out[0] = int32_t(around(at, taken, R));
        a.free_out[1] = int32_t(left - taken);
        a.free_out[2] = int32_t(min(want_all - taken + short_all, kPlanMost));
    }
    if (rows == 0) return;
    __threadfence_block();
    __syncthreads();
    for (uint32_t t = threadIdx.x; t < rows; t += kThreads) put_row_maps(a, page, t, find_seq(a.start, S, t));
}

__global__ __launch_bounds__(256) void k_plan_rows(tc_plan a, DivMod page) {
    const uint32_t t = blockIdx.x * 256 + threadIdx.x, first = blockIdx.x * 256;
    int seq = wave_find_seq(a.start, a.n_seq, first);
    const int32_t end = seq >= 0 ? a.start[seq + 1] : 0;
    if (t >= a.n_tokens) return;
    if (int32_t(t) >= end) seq = find_seq(a.start, a.n_seq, t);
    put_row_maps(a, page, t, seq);
}

constexpr uint32_t kRowsHere = 4096;

}  // namespace

hipError_t launch_plan(const tc_plan &p, hipStream_t st) {
    const DivMod page = make_divmod(p.page_tokens);
    const bool maps = p.sequence || p.position || p.slot;
    const bool here = maps && p.n_tokens <= kRowsHere;
    k_plan<<<1, kThreads, 0, st>>>(p, page, here ? p.n_tokens : 0);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !maps || here) return e;
    k_plan_rows<<<(p.n_tokens + 255) / 256, 256, 0, st>>>(p, page);
    return hipGetLastError();
}

}  // namespace tc
