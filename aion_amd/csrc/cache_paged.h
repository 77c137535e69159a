// Key/value caches in pages: the layout and the checks that every step over one makes (cache_paged.hip, cache_evict.hip, attention_paged.hip).
//
// Two pools [pages][H][P][D] of f16 or bf16, keys and values, and a table [B][W] of i32: step t of sequence b is row t % P of page table[b][t / P]. A head's rows
// of a page are one run, since a step reads one head's keys in order. P is a power of two from 16 on, so that sixteen neighbouring keys, what one matrix
// instruction takes, are rows of one page. An entry outside [0, pages) is no page: a kernel compares every entry it reads, what lies there is neither read nor written.
#pragma once
#include "common.h"

namespace paged {

constexpr size_t MIN_PAGE = 16, MAX_PAGE = 1024, MAX_HEAD = 1024, MAX_ROWS = 0x7FFFFFC0, MAX_THREADS = 0xFFFFFFFF;      // (of a launch, along one axis of its grid)

struct Table {
    const int *pages;
    int width, count, shift;      // entries of a sequence, pages of the pools, log2 of the rows of a page
};
// the page of a step, or -1
__device__ __forceinline__ int page_of(const Table &t, size_t b, int step) {
    const int e = step >> t.shift;
    if (step < 0 || e >= t.width) return -1;
    const int id = t.pages[b * (size_t)t.width + (size_t)e];
    return (unsigned)id < (unsigned)t.count ? id : -1;
}

inline int shift_of(size_t page_rows) { return __builtin_ctzll(page_rows); }
inline size_t capacity(const aionhip_paged_cache *c) { return c->table_width * c->page_rows; }
inline size_t pool_bytes(const aionhip_paged_cache *c) { return c->pages * c->h_kv * c->page_rows * c->d * 2; }
inline Table table_of(const aionhip_paged_cache *c) { return Table{(const int *)(uintptr_t)c->page_table, (int)c->table_width, (int)c->pages, shift_of(c->page_rows)}; }

inline bool overlap(aionhip_handle a, size_t a_bytes, aionhip_handle b, size_t b_bytes) { return a && b && a_bytes && b_bytes && a < b + b_bytes && b < a + a_bytes; }
// whether [h, h + bytes) lies in a pool or the table of the cache
inline bool in_cache(const aionhip_paged_cache *c, aionhip_handle h, size_t bytes) {
    return overlap(h, bytes, c->k_pages, pool_bytes(c)) || overlap(h, bytes, c->v_pages, pool_bytes(c)) || overlap(h, bytes, c->page_table, c->batch * c->table_width * 4);
}

inline int check_cache(aionhip_ctx *ctx, const char *who, const aionhip_paged_cache *c) {
    if (!c) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "%s: no cache", who);
    if (!c->k_pages || !c->v_pages || !c->page_table) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "%s: a cache has pools of keys and values and a page table", who);
    if (c->dtype != AIONHIP_F16 && c->dtype != AIONHIP_BF16) return set_err(ctx, AIONHIP_UNSUPPORTED, "%s: pages hold f16 or bf16, not dtype %d", who, c->dtype);
    if (c->page_rows < MIN_PAGE || c->page_rows > MAX_PAGE || (c->page_rows & (c->page_rows - 1)))
        return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "%s: a page has a power of two of rows, 16 to 1024, not %zu", who, c->page_rows);
    if (!c->pages || !c->table_width || !c->h_kv || !c->d) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "%s: a cache without pages, table entries, heads or columns", who);
    if (c->d % 8 != 0) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "%s: head size %zu is not a multiple of 8", who, c->d);
    if (c->d > MAX_HEAD || c->h_kv > 65535 || c->batch > 65535 || c->pages > 0x7FFFFFFF || c->table_width > MAX_ROWS / c->page_rows ||
        c->h_kv * c->page_rows * c->d > 0x3FFFFFFF)
        return set_err(ctx, AIONHIP_UNSUPPORTED, "%s: dimension too large", who);
    if ((c->k_pages | c->v_pages) & 15) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "%s: a pool begins at a multiple of 16 bytes", who);
    if (c->page_table & 3) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "%s: a page table begins at a multiple of 4 bytes", who);
    if (overlap(c->k_pages, pool_bytes(c), c->v_pages, pool_bytes(c))) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "%s: the pools of keys and values overlap", who);
    return AIONHIP_OK;
}

}  // namespace paged
