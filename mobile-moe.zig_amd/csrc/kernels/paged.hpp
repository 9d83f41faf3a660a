// Where a cached position's row lies in the paged pool, for the device and
// for the host (no HIP needed): every index that comes from device data is
// checked here, so that no page table, slot or length leads out of the pool.
#pragma once

#include <stdint.h>

#if defined(__HIP__) || defined(__HIPCC__)
#define MMHIP_HD __host__ __device__ __forceinline__
#else
#define MMHIP_HD inline
#endif

namespace mmhip {

struct PagedGeom {
    uint32_t width;       // values per row: rank + rope_dims
    uint32_t rank;
    uint32_t page_shift;  // log2(page_tokens)
    uint32_t n_pages;
    uint32_t q8;          // 1: i8 codes, then f16 block scales, per page
    uint64_t page_bytes;
};

// Pages of page_tokens rows: f16 values, or codes and then scales.
MMHIP_HD uint64_t paged_page_bytes(bool q8, uint32_t width, uint32_t page_tokens) {
    return (uint64_t)page_tokens * (q8 ? width + width / 32 * 2 : width * 2);
}

// Byte offset of a row's values (f16 values or codes), or of its scales.
MMHIP_HD uint64_t paged_row(const PagedGeom& g, uint32_t page, uint32_t at) {
    return page * g.page_bytes + (uint64_t)at * (g.q8 ? g.width : 2 * g.width);
}
MMHIP_HD uint64_t paged_scales(const PagedGeom& g, uint32_t page, uint32_t at) {
    return page * g.page_bytes + ((uint64_t)g.width << g.page_shift) + (uint64_t)at * (g.width / 32 * 2);
}

// A slot names a row of the pool; false: none (negative slots are skips).
MMHIP_HD bool paged_slot(const PagedGeom& g, int32_t slot, uint32_t& page, uint32_t& at) {
    page = (uint32_t)slot >> g.page_shift;
    at = (uint32_t)slot & ((1u << g.page_shift) - 1);
    return slot >= 0 && page < g.n_pages;
}

// Whether the pool has the page that a table entry names.
MMHIP_HD bool paged_has(const PagedGeom& g, int32_t id) { return id >= 0 && (uint32_t)id < g.n_pages; }

// Positions that a token sees: its length, at most what its table names; none
// where the table row does not exist. `bad`: 1 row, 2 length (0: neither).
MMHIP_HD uint32_t paged_seen(const PagedGeom& g, uint32_t len, uint32_t row, uint32_t n_tables, uint32_t table_pages,
                             uint32_t& bad) {
    bad = 0;
    if (row >= n_tables) {
        bad = 1;
        return 0;
    }
    const uint64_t most = (uint64_t)table_pages << g.page_shift;
    if (len > most) {
        bad = 2;
        return (uint32_t)most;
    }
    return len;
}

}  // namespace mmhip
