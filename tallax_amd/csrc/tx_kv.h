// A paged key-value cache as the kernels see it: slot s of sequence b lies in
// page table[b][s / page_size], at place s % page_size of each head.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "tallax_hip.h"
#include "tx_host.h"

namespace tx {

// Division of a slot number by the page size: n * mul >> shift is exact for
// 0 <= n < 2^31 (mul = floor(2^shift / d) + 1 with shift = 31 + ceil(log2 d),
// so mul * d - 2^shift <= d <= 2^(shift - 31), and mul fits 32 bits).
struct PageDiv {
  uint32_t mul;
  int shift;
  int size;
};

inline PageDiv make_page_div(int64_t d) {
  int s = 0;
  while (((int64_t)1 << s) < d) ++s;
  PageDiv p;
  p.shift = 31 + s;
  p.mul = (uint32_t)((((uint64_t)1 << p.shift) / (uint64_t)d) + 1);
  p.size = (int)d;
  return p;
}

__device__ __forceinline__ uint32_t page_of(const PageDiv& p, uint32_t slot) {
  return (uint32_t)(((uint64_t)slot * p.mul) >> p.shift);
}

struct KvView {
  char* k;
  char* v;
  int64_t k_page, k_head, k_slot;  // strides in bytes
  int64_t v_page, v_head, v_slot;
  const int32_t* table;
  int width;     // entries of a table row
  int capacity;  // slots a table row can hold
  int pages;
  int dim;
  PageDiv div;
};

// Checks a cache and turns it into a KvView (0 or a Status, with the message set).
int make_kv_view(const tallax_kv_cache* c, const char* what, KvView* out);

// The pool's page that holds `slot` of a sequence, -1 where the table names no page of the pool.
__device__ __forceinline__ int page_id(const KvView& c, const int32_t* row, int slot) {
  const int p = row[page_of(c.div, (uint32_t)slot)];
  return (uint32_t)p < (uint32_t)c.pages ? p : -1;
}

}  // namespace tx
