// Host-side pieces shared by the entry points on a paged cache.
#pragma once

#include "../../include/flash_prologue.h"
#include "gqa_rows.cuh"

namespace flash_prologue {

// Sizes, pointers and alignment of a cache (elements of `es` bytes) and its tables (status code).
int check_cache(const flash_prologue_cache& c, int64_t tokens, size_t es);
// Pointers and alignment of a 4-bit cache's scales.
int check_scales(const flash_prologue_scales& s, const flash_prologue_cache& c, int64_t D);

inline PagedTarget paged_target(const flash_prologue_cache& c) {
  PagedTarget t{};
  t.page_table = c.page_table;
  t.seq_lens = c.seq_lens;
  t.cu_seqlens = c.cu_seqlens;
  t.table_stride = c.table_stride;
  t.max_pages = c.max_pages;
  t.num_pages = c.num_pages;
  t.batch = (int)c.batch;
  while ((int64_t(1) << t.page_log2) < c.page_size) ++t.page_log2;
  return t;
}

}  // namespace flash_prologue
