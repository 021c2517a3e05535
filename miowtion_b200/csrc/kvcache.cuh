// The paged key-value cache: its storage formats and the address of a row.
//
// Pages are [n_pages, kv_heads, page_size, D]: the rows of one head lie
// together in a page, so a run of keys of a head is one contiguous piece.
// int8 and e4m3 rows carry one fp32 scale each, [n_pages, kv_heads,
// page_size]; a row is its codes times its scale.
#pragma once

#include "common.cuh"

namespace veda {

// Storage formats (the C ABI's numbers).
constexpr int kStoreBf16 = 0, kStoreInt8 = 1, kStoreE4m3 = 2;

struct CacheView {
  uint8_t* k;
  uint8_t* v;
  float* k_scale;  // null for bf16
  float* v_scale;
  int n_pages;
  int page_shift;  // page_size == 1 << page_shift
  int kv_heads;
  const int32_t* table;  // [n_seqs][table_ld] page numbers
  int64_t table_ld;
  int max_pages;  // entries of a table row
  int n_seqs;
};

// Host checks shared by the entry points; fills `view`.
int make_cache_view(CacheView* view, void* k, void* v, float* k_scale,
                    float* v_scale, int64_t n_pages, int32_t page_size,
                    int32_t kv_heads, int32_t head_dim, int32_t storage,
                    const int32_t* table, int64_t table_ld, int64_t max_pages,
                    int64_t n_seqs);

// Row index (in rows of D elements, and of the scales) of key `pos` of
// sequence `b`, head `h`; -1 when the table names no page of the cache.
__device__ __forceinline__ int64_t cache_row(const CacheView& c, int b, int h,
                                             int64_t pos) {
  const int64_t entry = pos >> c.page_shift;
  if (pos < 0 || entry >= c.max_pages) return -1;
  const int page = c.table[b * c.table_ld + entry];
  if (page < 0 || page >= c.n_pages) return -1;
  return (((static_cast<int64_t>(page) * c.kv_heads + h) << c.page_shift) |
          (pos & ((1 << c.page_shift) - 1)));
}

}  // namespace veda
