// The paged cache's host checks and page lookup, shared by the append and the
// attention over it.
#pragma once

#include "serving_checks.hpp"

namespace fh {

// Sizes of a paged cache: at least one page, pages of whole 16-key groups, and
// positions that fit 31 bits.
inline int check_pages(const char *fn, int64_t n_pages, int64_t page_size, int64_t max_pages) {
    if (n_pages < 1 || max_pages < 1)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: a paged cache has at least one page (n_pages %lld, max_pages %lld)",
                    fn, (long long)n_pages, (long long)max_pages);
    if (page_size < 16 || page_size % 16 != 0)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: page_size %lld must be a multiple of 16", fn, (long long)page_size);
    if (max_pages * page_size > 0x7FFFFFFFll)
        return fail(FH_ERR_INDEX_TOO_LARGE, "%s: max_pages * page_size exceeds 2^31 - 1", fn);
    return FH_OK;
}

// The K and V pools and the page table as operands of dev.
inline int check_pools(const fh_device *dev, const char *fn, const void *k_pages, const void *v_pages, int64_t n_pages,
                       int64_t n_kv, int64_t page_size, int64_t head_dim, const uint32_t *page_table, int64_t n_seqs,
                       int64_t max_pages, uint64_t *pool_bytes) {
    if ((reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages)) & 15u)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: pools must be 16-byte aligned", fn);
    uint64_t pool, table;
    if (int rc = size_product(fn, "a pool",
                              {static_cast<uint64_t>(n_pages), static_cast<uint64_t>(n_kv),
                               static_cast<uint64_t>(page_size), static_cast<uint64_t>(head_dim) * 2},
                              &pool))
        return rc;
    if (int rc = size_product(fn, "page_table", {static_cast<uint64_t>(n_seqs), static_cast<uint64_t>(max_pages), 4},
                              &table))
        return rc;
    if (int rc = check_range(dev, k_pages, pool, fn, "k_pages")) return rc;
    if (int rc = check_range(dev, v_pages, pool, fn, "v_pages")) return rc;
    *pool_bytes = pool;
    return check_range(dev, page_table, table, fn, "page_table");
}

}  // namespace fh
