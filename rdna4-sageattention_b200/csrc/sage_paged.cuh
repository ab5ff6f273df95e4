// The paged K/V cache as the kernels see it (layouts: include/sage_b200.h).
#pragma once

#include "sage_ptx.cuh"
#include "sage_rows.cuh"

namespace sage {

struct PagedArgs {
  int8_t* k8;          // [num_pages, Hkv, page_size, D]
  float* ks;           // [num_pages, Hkv, page_size]
  uint8_t* v8;         // e4m3, as k8
  float* vs;
  int num_pages, page_shift, Hkv, D;
  const int* table;    // [B, max_pages]
  int64_t table_stride;
  int max_pages;
  const int* lens;     // [B]
  int* status;
};

__device__ __forceinline__ void raise_invalid(const PagedArgs& p) { *const_cast<volatile int*>(p.status) = kStatusInvalid; }

// Row number (page * Hkv + head) * page_size + offset of position `at` of sequence b, or -1 (and the status word
// set) where the table has no valid page for it.
__device__ __forceinline__ int64_t paged_row(const PagedArgs& p, int b, int head, int64_t at) {
  const int64_t slot = at >> p.page_shift;
  if (at < 0 || slot >= p.max_pages) {
    raise_invalid(p);
    return -1;
  }
  const int page = p.table[b * p.table_stride + slot];
  if (page < 0 || page >= p.num_pages) {
    raise_invalid(p);
    return -1;
  }
  return ((((int64_t)page * p.Hkv + head) << p.page_shift) + (at & ((1 << p.page_shift) - 1)));
}

// Host side: the cache arguments of an entry point, checked.
int paged_args(PagedArgs* out, void* k8, float* ks, void* v8, float* vs, int num_pages, int page_size, int Hkv, int D,
               const int32_t* page_table, int64_t table_stride, int max_pages, const int32_t* lens, int* status);

}  // namespace sage
