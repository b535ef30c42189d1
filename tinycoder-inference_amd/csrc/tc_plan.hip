// tc_plan.hip -- the geometry of a step from its sequences' lengths.
//
// Sums over the sequences in their order decide everything: rows, and pages given back, then
// pages wanted, which depend on the rows. One workgroup forms them, as many sequences at a time
// as it has threads, and enters the pages, a thread a page whosever it is; with that done, a row's
// sequence, position and slot are looked up as the other kernels do. Few rows are looked up by the
// same workgroup, with the sequences' starts in LDS (1200 rows 4.8 us, 5.7 with a launch of their own;
// 4000 rows 6.0 and 5.8).
// Bound by the chain lengths -> sums -> ring -> table -> slots, not by any traffic.
//
// Sums of rows saturate at n_tokens, and those of missing pages at 2^30, so that they stay in 32
// bits whatever the arrays hold; min(a + b, top) is associative for numbers that are not negative.
// The others are at most the tables' entries, 2^30.
#include "tc_kernels.hpp"
#include "tc_step.hpp"

namespace tc {
namespace {

// What stands N lanes to the left and the like (DPP); 0 where there is none.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t left_lane(uint32_t v) {
    return uint32_t(__builtin_amdgcn_update_dpp(0, int(v), CTRL, ROWS, 15, false));
}
// The wave's sums up to each lane, saturating at top. All lanes call it.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v, uint32_t top) {
    v = min(v + left_lane<0x111, 15>(v), top);  // 1, 2, 4, 8 lanes to the left in rows of 16
    v = min(v + left_lane<0x112, 15>(v), top);
    v = min(v + left_lane<0x114, 15>(v), top);
    v = min(v + left_lane<0x118, 15>(v), top);
    v = min(v + left_lane<0x142, 10>(v), top);  // the last lane of rows 0 and 2 to rows 1 and 3
    v = min(v + left_lane<0x143, 12>(v), top);  // lane 31 to rows 2 and 3
    return v;
}

struct Sum {
    uint32_t before, all;  // over the threads before this one, over all
};
// Two sums over a workgroup of THREADS, the first saturating at top0, the second at top1. lds:
// a place that no other scan uses but the one before the last. Every thread calls it.
template <int THREADS>
__device__ __forceinline__ void block_scan(uint32_t v0, uint32_t top0, uint32_t v1, uint32_t top1, uint32_t (&lds)[2][THREADS / 64],
                                           Sum &s0, Sum &s1) {
    constexpr uint32_t WAVES = THREADS / 64;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t a = wave_scan(v0, top0), b = wave_scan(v1, top1);
    if (lane == 63) lds[0][wave] = a, lds[1][wave] = b;
    __syncthreads();
    const uint32_t wa = wave_scan(lane < WAVES ? lds[0][lane] : 0, top0), wb = wave_scan(lane < WAVES ? lds[1][lane] : 0, top1);
    const uint32_t ba = wave ? __builtin_amdgcn_readlane(wa, wave - 1) : 0, bb = wave ? __builtin_amdgcn_readlane(wb, wave - 1) : 0;
    // (each lane's sum without its own: the lane's to the left)
    s0 = {min(ba + uint32_t(__shfl_up(int(a), 1)) * (lane != 0), top0), uint32_t(__builtin_amdgcn_readlane(wa, WAVES - 1))};
    s1 = {min(bb + uint32_t(__shfl_up(int(b), 1)) * (lane != 0), top1), uint32_t(__builtin_amdgcn_readlane(wb, WAVES - 1))};
}

__device__ __forceinline__ uint32_t bounded(int32_t v, uint32_t most) { return v < 0 ? 0u : min(uint32_t(v), most); }
// Place of the ring, `by` (up to 2^30) from place `at` on.
__device__ __forceinline__ uint32_t around(uint32_t at, uint32_t by, uint32_t ring) {
    uint32_t i = at + by;  // (ring, at and by are at most 2^30)
    if (i >= ring) i -= ring;
    return i >= ring ? i % ring : i;
}

// Half of the least power of two that n (at least 1) is not above.
__device__ __forceinline__ uint32_t first_step(uint32_t n) { return n <= 1 ? 0 : 1u << (31 - __builtin_clz(n - 1)); }
// Of an ascending list the last entry that is at most v (list[0] is), among as many as `first` is the
// first step of, and those up to twice that.
__device__ __forceinline__ uint32_t find_last(const uint32_t *list, uint32_t first, uint32_t v) {
    uint32_t at = 0;
    for (uint32_t step = first; step != 0; step /= 2) at += list[at + step] <= v ? step : 0;
    return at;
}
// put(j, i, get(j, i)) for the pages j < n of a lot of sequences, i the sequence's place in it. Where
// there are more pages than threads, a thread's next four side by side: each one's search and
// fetch are a chain of their own.
template <uint32_t THREADS, class Get, class Put>
__device__ __forceinline__ void each_page(const uint32_t *before, uint32_t first, uint32_t n, Get get, Put put) {
    uint32_t j0 = threadIdx.x;
    for (; j0 + 3 * THREADS < n; j0 += 4 * THREADS) {
        uint32_t i[4];
        int32_t v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) i[k] = 0;
        for (uint32_t step = first; step != 0; step /= 2)
#pragma unroll
            for (int k = 0; k < 4; ++k) i[k] += before[i[k] + step] <= j0 + k * THREADS ? step : 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = get(j0 + k * THREADS, i[k]);
#pragma unroll
        for (int k = 0; k < 4; ++k) put(j0 + k * THREADS, i[k], v[k]);
    }
    for (; j0 < n; j0 += THREADS) {
        const uint32_t i = find_last(before, first, j0);
        put(j0, i, get(j0, i));
    }
}

// A row's sequence (-1: none), position (below 0: none, where a length was held to the largest)
// and slot.
__device__ __forceinline__ void put_row_maps(const tc_plan &a, const DivMod &page, uint32_t t, int seq, int32_t pos) {
    int64_t slot = -1;
    if (pos >= 0) {
        const uint32_t pi = div_fast(uint32_t(pos), page);
        if (pi < a.table_pages) {
            const int32_t pg = a.table[size_t(seq) * a.table_pages + pi];
            if (pg >= 0) slot = int64_t(pg) * a.page_tokens + (uint32_t(pos) - pi * a.page_tokens);
        }
    } else {
        pos = -1;
    }
    if (a.sequence) a.sequence[t] = seq;
    if (a.position) a.position[t] = pos;
    if (a.slot) a.slot[t] = slot;
}
__device__ __forceinline__ int32_t position_of(const tc_plan &a, uint32_t t, int seq) {
    return seq < 0 ? -1 : a.len[seq] - a.start[seq + 1] + int32_t(t);
}

template <int THREADS>
__global__ __launch_bounds__(THREADS) void k_plan(tc_plan a, DivMod page, uint32_t rows) {
    __shared__ uint32_t sums[2][2][THREADS / 64];
    __shared__ uint32_t before[THREADS], had_of[THREADS], begins[THREADS];
    __shared__ int32_t shift[THREADS];  // of a sequence's rows to their positions
    const uint32_t S = a.n_seq, R = a.ring_pages, W = a.table_pages, tid = threadIdx.x;
    const uint32_t at = bounded(a.free[0], R - 1), left0 = bounded(a.free[1], R);
    const uint32_t first = first_step(min(S, uint32_t(THREADS)));  // of searches among a lot of sequences
    int turn = 0;
    // pages of ended sequences behind the free ones, and where there is one lot of sequences only, their rows
    uint32_t back_all = 0, row_all = 0;
    Sum rows_of{0, 0}, back_of, none;
    int32_t fresh = -1;
    uint32_t held = 0, had = 0;
    auto fetch = [&](uint32_t s) {
        fresh = s < S ? a.new_tokens[s] : -1;
        held = s < S ? bounded(a.held[s], kLenMost) : 0;
        had = s < S ? bounded(a.pages[s], W) : 0;
    };
    for (uint32_t s0 = 0; s0 < S; s0 += THREADS) {
        fetch(s0 + tid);
        const uint32_t back = fresh < 0 ? had : 0;
        block_scan<THREADS>(back, kPlanMost, bounded(fresh, a.n_tokens), a.n_tokens, sums[turn ^= 1], back_of, rows_of);
        if (back_of.all != 0) {  // a thread a page
            before[tid] = back_of.before;
            __syncthreads();
            const uint32_t room = left0 + back_all < R ? R - left0 - back_all : 0;
            each_page<THREADS>(
                before, first, min(back_of.all, room), [&](uint32_t j, uint32_t i) { return a.table[size_t(s0 + i) * W + (j - before[i])]; },
                [&](uint32_t j, uint32_t, int32_t page) { a.ring[around(at, left0 + back_all + j, R)] = page; });
            __threadfence_block();
            __syncthreads();
        }
        back_all += back_of.all;
    }
    const uint32_t left = min(left0 + back_all, R);
    uint32_t want_all = 0, short_all = 0;
    for (uint32_t s0 = 0; s0 < S; s0 += THREADS) {
        const uint32_t s = s0 + tid;
        if (S > THREADS) {
            fetch(s);
            block_scan<THREADS>(bounded(fresh, a.n_tokens), a.n_tokens, 0, 0, sums[turn ^= 1], rows_of, none);
        }
        const uint32_t begin = min(row_all + rows_of.before, a.n_tokens);
        row_all = min(row_all + rows_of.all, a.n_tokens);
        const uint32_t got_rows = min(bounded(fresh, a.n_tokens), a.n_tokens - begin);
        const uint32_t len = fresh < 0 ? 0 : min(held + got_rows, uint32_t(kLenMost));
        uint32_t need = div_fast(len, page);
        if (need * a.page_tokens < len) ++need;
        const uint32_t fit = min(need, W), want = fresh >= 0 && fit > had ? fit - had : 0;
        Sum want_of, short_of;
        block_scan<THREADS>(want, kPlanMost, need - fit, kPlanMost, sums[turn ^= 1], want_of, short_of);
        if (s < S) {
            const uint32_t from = want_all + want_of.before;
            a.start[s] = int32_t(begin);
            a.len[s] = int32_t(len);
            a.pages_out[s] = fresh < 0 ? 0 : int32_t(had + (from < left ? min(want, left - from) : 0));
        }
        begins[tid] = begin;
        shift[tid] = int32_t(len) - int32_t(begin + got_rows);
        if (want_of.all != 0) {  // a thread a page
            before[tid] = want_of.before;
            had_of[tid] = had;
            __syncthreads();
            each_page<THREADS>(
                before, first, want_of.all, [&](uint32_t j, uint32_t) { return want_all + j < left ? a.ring[around(at, want_all + j, R)] : -1; },
                [&](uint32_t j, uint32_t i, int32_t page) { a.table[size_t(s0 + i) * W + had_of[i] + (j - before[i])] = page; });
            __syncthreads();
        }
        want_all += want_of.all;
        short_all = min(short_all + short_of.all, kPlanMost);
    }
    if (tid == 0) {
        const uint32_t taken = min(want_all, left);
        a.start[S] = int32_t(row_all);
        a.free_out[0] = int32_t(around(at, taken, R));
        a.free_out[1] = int32_t(left - taken);
        a.free_out[2] = int32_t(min(want_all - taken + short_all, kPlanMost));
    }
    if (rows == 0) return;
    __threadfence_block();
    __syncthreads();
    for (uint32_t t = tid; t < rows; t += THREADS) {
        int seq = -1;
        int32_t pos = -1;
        if (t < row_all) {
            seq = S > THREADS ? find_seq(a.start, S, t) : int(find_last(begins, first, t));
            pos = S > THREADS ? position_of(a, t, seq) : shift[seq] + int32_t(t);
        }
        put_row_maps(a, page, t, seq, pos);
    }
}

// The rows' maps, a row a thread. Up to 1024 sequences' starts are held in LDS: one fetch and a
// search there, where each step of a search in memory waits for the one before (301 sequences with 165000
// rows, both launches, 9.9 us where that took 10.7).
constexpr uint32_t kSeqsHere = 1024;
__global__ __launch_bounds__(256) void k_plan_rows(tc_plan a, DivMod page) {
    __shared__ uint32_t begins[kSeqsHere];
    __shared__ int32_t shift[kSeqsHere];
    const uint32_t S = a.n_seq, t = blockIdx.x * 256 + threadIdx.x, first = first_step(S);
    const uint32_t all = uint32_t(a.start[S]);
    if (S <= kSeqsHere) {
        // (entries behind the last sequence that a search looks at are above every row)
        for (uint32_t s = threadIdx.x; s < max(S, 2 * first); s += 256) {
            begins[s] = s < S ? uint32_t(a.start[s]) : ~0u;
            shift[s] = s < S ? a.len[s] - a.start[s + 1] : 0;
        }
        __syncthreads();
    }
    if (t >= a.n_tokens) return;
    int seq = -1;
    int32_t pos = -1;
    if (t < all) {
        seq = S > kSeqsHere ? find_seq(a.start, S, t) : int(find_last(begins, first, t));
        pos = S > kSeqsHere ? position_of(a, t, seq) : shift[seq] + int32_t(t);
    }
    put_row_maps(a, page, t, seq, pos);
}

constexpr uint32_t kRowsHere = 4096;

}  // namespace

hipError_t launch_plan(const tc_plan &p, hipStream_t st) {
    const DivMod page = make_divmod(p.page_tokens);
    const bool maps = p.sequence || p.position || p.slot;
    const bool here = maps && p.n_tokens <= kRowsHere;
    const uint32_t rows = here ? p.n_tokens : 0;
    // (barriers of 4 waves cost less than those of 16, 32 sequences of a row each 4.2 us and 4.8, and one wave
    // has none: 3.9; many rows and pages want the threads, 256 rows 5.8 with 64, 4.3 with 256 and 4.8 with
    // 1024, 800 rows 5.0 with 256 and 4.6 with 1024. Pages alone, of 4000 rows, 5.8 with 256 and 6.4 with
    // 1024, of 12000 7.3 and 6.7)
    if (p.n_seq <= 64 && here && rows <= 64)
        k_plan<64><<<1, 64, 0, st>>>(p, page, rows);
    else if (p.n_seq <= 256 && (here ? rows <= 512 : p.n_tokens <= 8192))
        k_plan<256><<<1, 256, 0, st>>>(p, page, rows);
    else
        k_plan<1024><<<1, 1024, 0, st>>>(p, page, rows);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !maps || here) return e;
    k_plan_rows<<<(p.n_tokens + 255) / 256, 256, 0, st>>>(p, page);
    return hipGetLastError();
}

}  // namespace tc
