// nkv_paged.h -- types shared by the kernels of the paged key/value cache
// (nkv_paged.hip, nkv_paged_attend.hip).
//
// A pool holds pages of `page` rows (a power of two, 16 at least) of every key
// head, [pages, H, page, D] in 16 bits; a table names each sequence's pages in
// order.  An entry outside [0, pages) names no page.
#pragma once

#include "nkv_cache8.h"

namespace nkv {

// A page table in device memory and what is needed to find a row with it.
struct PageTable {
    const int32_t* at;            // [B][w], sb apart
    int64_t sb, w;
    uint32_t pages;
    int shift;                    // log2 of a page's rows
    int64_t page_elems;           // elements of a page in all heads
    // rows that item tables have room for
    __host__ __device__ __forceinline__ int64_t cap() const { return w << shift; }
};

// Element of row `row` of a sequence (in its head 0's part of the page), or -1 where
// the row lies outside the table or in no page.
__device__ __forceinline__ int64_t page_row(const PageTable& t, int b, int64_t row, int D) {
    if (row < 0 || row >= t.cap()) return -1;
    const uint32_t id = (uint32_t)t.at[b * t.sb + (row >> t.shift)];
    if (id >= t.pages) return -1;
    return (int64_t)id * t.page_elems + (row & ((1 << t.shift) - 1)) * D;
}

// The first row of batch item b's new rows.
__device__ __forceinline__ int64_t paged_start(const int32_t* start_dev, int b, int64_t start,
                                               int64_t cap) {
    if (!start_dev) return start;
    const int64_t s = start_dev[b];
    return s < 0 ? 0 : s < cap ? s : cap;
}

// Validates a cache, and a table of it (host).
int paged_check(const nkv_paged_cache& c, const char* who);
int paged_table_check(const nkv_paged_cache& c, const int32_t* table, int64_t sb, int64_t w, int B,
                      const char* who);
PageTable page_table(const nkv_paged_cache& c, const int32_t* table, int64_t sb, int64_t w);

// Bytes of one pool, and of a table.
inline int64_t pool_bytes(const nkv_paged_cache& c) { return c.pages * c.H * c.page * c.D * 2; }
inline int64_t table_bytes(int B, int64_t sb, int64_t w) { return B ? ((B - 1) * sb + w) * 4 : 0; }

// The elements that rows of n0 x n1 x n2 (strides s0, s1, s2) of D span, or -1 where
// two of them overlap (or a stride is negative).
int64_t rows_span(int64_t s0, int64_t n0, int64_t s1, int64_t n1, int64_t s2, int64_t n2, int D);

// Rows of `bytes` bytes, some of them or none (bytes = 0), at `at` + multiples of three
// strides, in bytes; they lie in the `span` bytes from there on (host).
struct RowSet {
    uintptr_t at = 0;
    int64_t bytes = 0;
    __int128 span = 0;
    struct {
        int64_t stride = 0, count = 1;
    } dims[3];
    // strides of elements of es bytes, not negative; none where p is null
    RowSet(const void* p, int es, int D, int64_t s0, int64_t n0, int64_t s1, int64_t n1, int64_t s2, int64_t n2);
    RowSet(const Range& r) : at(r.lo), bytes((int64_t)(r.hi - r.lo)), span(bytes) {}
};

// Whether two sets have a byte in common.  Exact for rows that do not overlap within their
// set where one set has no gaps, or both have the same strides (slices of one projection);
// rows that do overlap are taken for all that they span, and others of unlike strides, both
// with gaps, for apart.
bool rows_meet(const RowSet& a, const RowSet& b);

}  // namespace nkv
