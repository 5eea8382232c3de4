// Slots of a paged per-head cache in TurboQuant codes, shared by the kernels that write, attend and shrink it.
//
// A pool holds `pages` pages of [heads, page_size, row] codes and [heads, page_size] fp32 scales, for K and for V.
// Sequence b's slot p lies in row p % page_size of page table[b, p / page_size].  Lengths, starts and tables are device
// data that the host cannot check, so every use goes through these functions: a slot outside the table, or a page outside
// the pool, has no address and is skipped, as the attention kernels skip a selected index outside the cache.
#pragma once

#include "aekv_common.h"
#include "paged_slot.h"

namespace aekv {

// Host-side checks shared by the entry points; fills the pool.  AEKV_OK or the failure.
int check_pool(const char* who, void* k_codes, float* k_scale, void* v_codes, float* v_scale, int64_t pages,
               int64_t heads, int32_t page_size, int32_t d, int32_t bits, const int32_t* table, int64_t max_pages,
               int64_t B, PagePool* out);

}  // namespace aekv
