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

// x / d as (x * mul) >> shift for x below 2^26: mul = ceil(2^shift / d) with shift = 26 + ceil(log2 d),
// whose excess mul * d - 2^shift < d <= 2^(shift - 26) never reaches the next quotient.
struct PageDiv {
    uint32_t mul;
    int32_t shift;
};
inline PageDiv paged_div(int d) {
    int s = 0;
    while ((1 << s) < d) ++s;
    return {(uint32_t)((((uint64_t)1 << (26 + s)) + d - 1) / d), 26 + s};
}
KUIOPS_HOST_DEVICE int paged_quotient(int x, PageDiv d) { return (int)((uint64_t)(uint32_t)x * d.mul >> d.shift); }

// Which entry of its row of the table a slot (>= 0) has, and which row of that page; `div`
// divides by a page's 16-slot groups.  For 16 slots from a multiple of 16 on it is the same
// page, whose size is a multiple too.
KUIOPS_HOST_DEVICE int paged_entry(int slot, int page, PageDiv div, int &at) {
    const int p = paged_quotient(slot >> 4, div);
    at = slot - p * page;
    return p;
}

// The page of a slot (-1: none) and its row there.  Nothing outside the table's row is read.
KUIOPS_HOST_DEVICE int paged_find(const int32_t *row, int width, int page, PageDiv div, int pages, int slot, int &at) {
    const bool in = slot >= 0 && slot < width * page;
    const int p = paged_entry(in ? slot : 0, page, div, at);
    return in ? paged_id(row[p], pages) : -1;
}

// How many of the 16 slots from `slot` on are there.
KUIOPS_HOST_DEVICE int paged_rows16(int id, int slot, int end) {
    const int left = end - slot;
    return id < 0 || left < 0 ? 0 : left < 16 ? left : 16;
}

}  // namespace kuiops
