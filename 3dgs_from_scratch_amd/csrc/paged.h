// A paged cache's tables, as its kernels read them (see GsPages).
#pragma once

#include "element.h"

namespace gs {

constexpr int64_t kMaxSlots = 0x7fffffffLL - 65536;  // slot numbers stay in 32 bits

// The page of a sequence's slots from index * page_size on, or -1 where there is none.
__device__ __forceinline__ int page_of(const GsPages &p, int sequence, int index) {
    const int32_t page = p.tables[(int64_t)sequence * p.table_stride + index];
    return (uint32_t)page < (uint64_t)p.pages ? page : -1;
}

__device__ __forceinline__ int filled_slots(const GsPages &p, int sequence) {
    const int64_t most = (int64_t)p.page_size * p.table_width;
    const int n = p.lengths[sequence];
    return n < 0 ? 0 : n < most ? n : (int)most;
}

// a b in 64 bits, by one multiplication: the strides of a pool fit in 31 bits.
__device__ __forceinline__ int64_t times(int a, int64_t b) {
    return (int64_t)((uint64_t)(uint32_t)a * (uint32_t)b);
}

// First element of a slot's key or value of head 0, and its weight's.
__device__ __forceinline__ int64_t row_at(const GsPages &p, int page, int place) {
    return times(page, p.page_stride) + times(place, p.slot_stride);
}
__device__ __forceinline__ int64_t sum_at(const GsPages &p, int page, int place, int head) {
    return times(page, p.sum_page) + times(place, p.sum_slot) + times(head, p.sum_head);
}

// Status of a cache's description; nothing is launched where it is not GS_OK.
int check_pages(const GsPages *p, bool weights);

}  // namespace gs
