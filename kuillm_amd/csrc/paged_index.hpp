// Where the slots of a paged KV cache lie.  Nothing here needs HIP, so that the arithmetic
// that keeps a kernel inside the pool can be run on the host.
#pragma once

#include <stdint.h>

#if defined(__HIPCC__)
#define KUIOPS_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define KUIOPS_HOST_DEVICE inline
#endif

namespace kuiops {

// A sequence's slots: its length, as far as its row of the table goes.
KUIOPS_HOST_DEVICE int paged_slots(int len, int width, int page) {
    const int most = width * page;
    return len < 0 ? 0 : len < most ? len : most;
}

// An entry of the table that is no page of the pool is -1.
KUIOPS_HOST_DEVICE int paged_id(int entry, int pages) { return (unsigned)entry < (unsigned)pages ? entry : -1; }

// The page of a slot (-1: none) and its row there.  Nothing behind the table's row is read.
KUIOPS_HOST_DEVICE int paged_find(const int32_t *row, int width, int page, int pages, int slot, int &at) {
    const int p = slot / page;
    at = slot - p * page;
    return slot >= 0 && p < width ? paged_id(row[p], pages) : -1;
}

// The same for the 16 slots from `slot` on (a multiple of 16, pages are too), as long as some
// of them lie below `end` (at most the sequence's slots).
KUIOPS_HOST_DEVICE int paged_find16(const int32_t *row, int page, int pages, int slot, int end, int &at) {
    const int gpp = page / 16, g = slot / 16, p = g / gpp;
    at = (g - p * gpp) * 16;
    return slot >= 0 && slot < end ? paged_id(row[p], pages) : -1;
}

// How many of the 16 slots from `slot` on are there.
KUIOPS_HOST_DEVICE int paged_rows16(int id, int slot, int end) {
    const int left = end - slot;
    return id < 0 || left < 0 ? 0 : left < 16 ? left : 16;
}

}  // namespace kuiops
