// Where a slot of a paged cache lies (paged_cache.h).  Plain C++, so that a host compiler can check it.
#pragma once

#include <cstdint>

namespace aekv {

struct PagePool {
  uint8_t* k_codes;
  float* k_scale;
  uint8_t* v_codes;
  float* v_scale;
  const int32_t* table;  // [B, max_pages]
  int32_t pages, max_pages, heads, page_shift;  // page_size = 1 << page_shift, at least 16
};

// Slots the table has room for (the launchers check that they fit 31 bits).
__device__ __forceinline__ int32_t table_slots(const PagePool& c) { return c.max_pages << c.page_shift; }

// Row index ((page * heads + head) * page_size + row) of slot p of sequence b, or -1 where it has none.
__device__ __forceinline__ int64_t cache_row(const PagePool& c, int64_t b, int32_t head, int64_t p) {
  if (p < 0 || p >= table_slots(c)) return -1;
  const int32_t page = c.table[b * c.max_pages + (p >> c.page_shift)];
  if (page < 0 || page >= c.pages) return -1;
  return (((static_cast<int64_t>(page) * c.heads + head) << c.page_shift)) + (p & ((1 << c.page_shift) - 1));
}

}  // namespace aekv
