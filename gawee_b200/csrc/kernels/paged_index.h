// Where a sequence's cached row lies in the pages of a paged key/value cache.
// Plain C++, so that the index arithmetic can be checked without a GPU.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define GAWEE_HD __host__ __device__ __forceinline__
#else
#define GAWEE_HD inline
#endif

namespace gawee {
namespace kern {

// Pages [num_pages][kv_heads][page_size][row] of a K or a V cache; the page
// stride may be larger than a page (caches of several layers in one buffer).
struct PageGeom {
  int64_t page_stride;  // elements
  int64_t num_pages;
  int kv_heads, page_size, head_dim;
};

// log2 of a page size, -1 where it is no power of two.
inline int page_shift_of(int page_size) {
  for (int b = 0; b <= 16; ++b)
    if (page_size == 1 << b) return b;
  return -1;
}

// The page that holds row `pos` of the sequence whose block-table row is
// `table` (`cols` columns), or -1 where the table has no such column or names
// a page that does not exist.
GAWEE_HD int64_t page_of(const int32_t* table, int64_t cols, int64_t pos, const PageGeom& g) {
  if (pos < 0) return -1;
  const int64_t col = pos / g.page_size;
  if (col >= cols) return -1;
  const int32_t page = table[col];
  return page >= 0 && page < g.num_pages ? (int64_t)page : -1;
}

// Element offset of (page, head, slot) from the base of the pages: 64 bits,
// a long cache passes 2^31 elements.
GAWEE_HD int64_t row_offset(int64_t page, int head, int slot, const PageGeom& g) {
  return page * g.page_stride + ((int64_t)head * g.page_size + slot) * g.head_dim;
}

}  // namespace kern
}  // namespace gawee
