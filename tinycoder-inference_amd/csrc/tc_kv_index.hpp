// tc_kv_index.hpp -- the geometry of a batch over a paged cache: which rows are
// whose, and in which cache row a position lies. Every number that comes from the
// batch's arrays is bounded here, so that no value in them leads out of the cache,
// the page table or the call's rows. Plain C++: host programs can run it.
#pragma once

#include <stddef.h>
#include <stdint.h>

#ifdef __HIPCC__
#define TC_HD __host__ __device__ __forceinline__
#else
#define TC_HD inline
#endif

namespace tc {

// Fast unsigned division by a runtime constant (Granlund-Montgomery): q = n/d
// for n < 2^31, using the high half of a 32x32->64 multiply.
struct DivMod {
    uint32_t d, mul, shift;
};

inline DivMod make_divmod(uint32_t d) {
    DivMod r{d, 0, 0};
    uint32_t s = 0;
    while ((uint64_t(1) << s) < d) ++s;
    r.shift = s;
    // mul = ceil(2^(32+s) / d) - 2^32
    const uint64_t one = 1;
    r.mul = uint32_t(((one << 32) * ((one << s) - d)) / d + 1);
    return r;
}

TC_HD uint32_t div_fast(uint32_t n, const DivMod &m) {
    if (m.d == 1) return n;
    const uint32_t t = uint32_t((uint64_t(n) * m.mul) >> 32);
    return (t + ((n - t) >> 1)) >> (m.shift - 1);
}

// The cache and the batch of one call, by value.
struct KvArgs {
    uint8_t *k, *v;
    float *ks, *vs;
    uint32_t n_pages, kv_heads, page, dim;
    DivMod page_div;
    const int32_t *start, *len, *table;
    uint32_t n_seq, n_tokens, table_pages;
};

constexpr uint32_t kMaxPos = 0x7FFFFFFF;

// Row range of sequence s, kept inside the call's rows whatever start holds.
TC_HD void seq_rows(const int32_t *start, uint32_t n_tokens, uint32_t s, uint32_t *begin, uint32_t *end) {
    const int32_t T = int32_t(n_tokens), x = start[s], y = start[s + 1];
    const int32_t b = x < 0 ? 0 : x > T ? T : x;
    const int32_t e = y < b ? b : y > T ? T : y;
    *begin = uint32_t(b);
    *end = uint32_t(e);
}

// The sequence that row t belongs to (of those starting at or before it the
// last), -1 for rows past the last sequence or before the first.
TC_HD int find_seq(const int32_t *start, uint32_t n_seq, uint32_t t) {
    uint32_t lo = 0, hi = n_seq;  // start[lo] <= t < start[hi]
    if (int32_t(t) >= start[hi] || int32_t(t) < start[0]) return -1;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (start[mid] <= int32_t(t))
            lo = mid;
        else
            hi = mid;
    }
    return int(lo);
}

// Page of the pi-th page of sequence s; -1 where the table has none or an id
// outside the cache.
TC_HD int32_t page_at(const KvArgs &a, uint32_t s, uint32_t pi) {
    if (pi >= a.table_pages) return -1;
    const uint32_t pg = uint32_t(a.table[size_t(s) * a.table_pages + pi]);
    return pg < a.n_pages ? int32_t(pg) : -1;
}

// Cache row (page * kv_heads + head) * page_tokens + slot of batch row t of sequence s
// (-1: none) and head; a cache may have more than 2^31 rows. (No branch between the
// loads: a lane's rows are looked up side by side.)
TC_HD int64_t slot_of(const KvArgs &a, int s, uint32_t t, uint32_t head) {
    const uint32_t q = s < 0 ? 0 : uint32_t(s);
    const int64_t pos = int64_t(a.len[q]) - a.start[q + 1] + t;
    bool ok = s >= 0 && pos >= 0 && pos < int64_t(kMaxPos);
    const uint32_t p = ok ? uint32_t(pos) : 0, pi = div_fast(p, a.page_div);
    ok = ok && pi < a.table_pages;
    const uint32_t pg = uint32_t(a.table[size_t(q) * a.table_pages + (ok ? pi : 0)]);
    ok = ok && pg < a.n_pages;
    return ok ? (int64_t(pg) * a.kv_heads + head) * a.page + (p - pi * a.page) : -1;
}

}  // namespace tc
