// The paged KV cache as its kernels see it: a pool of pages that the sequences share,
// and a table per sequence that names its pages.
#pragma once

#include "common.hpp"
#include "paged_index.hpp"

namespace kuiops {

// Slot j of sequence b is row j % page of page table[b][j / page]; an entry outside
// 0 .. pages - 1 is no page.  Strides in elements of their tensor.
struct PagedCache {
    const void *K, *V;
    const float *ks, *vs;              // a scale per row of 8-bit pages
    const int32_t *table;
    int64_t sk0, sk1, sk2, sv0, sv1, sv2, sks0, sks1, svs0, svs1, ld_table;
    int pages, page, hkv, hd, width;
    PageDiv div;                       // by a page's 16-slot groups
    int dtype;
};

__device__ __forceinline__ int page_of(const PagedCache &c, int64_t b, int slot, int &at) {
    return paged_find(c.table + b * c.ld_table, c.width, c.page, c.div, c.pages, slot, at);
}

__device__ __forceinline__ int paged_len(const PagedCache &c, const int32_t *kv_len, int64_t b) {
    return paged_slots(kv_len[b], c.width, c.page);
}

// What every entry point asks of the cache; KUIOPS_OK if the kernels take it.
int check_cache(const kuiops_paged_layout *at, int dtype, const void *K, const void *V, const float *ks, const float *vs,
                const int32_t *table, PagedCache &c);

}  // namespace kuiops
