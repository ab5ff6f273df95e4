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

// Four int8 codes -> two fp16 pairs, exactly: 0x6400 + u is the fp16 number 1024 + u, and u = code + 128.
__device__ __forceinline__ void int8_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  w ^= 0x80808080u;
  const __half2 off = __half2half2(__ushort_as_half(0x6480));   // 1152
  uint32_t x = __byte_perm(w, 0x64646464u, 0x4140), y = __byte_perm(w, 0x64646464u, 0x4342);
  const __half2 p = __hsub2(*reinterpret_cast<__half2*>(&x), off), q = __hsub2(*reinterpret_cast<__half2*>(&y), off);
  lo = *reinterpret_cast<const uint32_t*>(&p);
  hi = *reinterpret_cast<const uint32_t*>(&q);
}

// Two e4m3 codes -> an fp16 pair (exact).
__device__ __forceinline__ uint32_t e4m3_to_f16(uint16_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
  return r;
}

// Host side: the cache arguments of an entry point, checked.
int paged_args(PagedArgs* out, const sage_paged_kv& kv);

}  // namespace sage
