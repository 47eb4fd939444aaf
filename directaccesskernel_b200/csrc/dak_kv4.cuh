// dak_kv4.cuh - the 4-bit paged KV cache's layout and page lookup.
//
// A pool is [pages, kv_heads, slab bytes]; one (page, head) slab of P tokens
// holds, one after the other,
//   K codes [P][64]                    (dim 2i in the low nibble of byte i)
//   K (scale, zero) [P][NG][2] float16 (NG = 128 / group)
//   V codes [P][64]
//   V (scale, zero) [P][NG][2] float16
// and the value of code n is scale * n + zero, scale >= 0.  K and V of a page sit in one
// slab so that one contiguous copy (2.1 to 10 KB) brings both.
#pragma once

#include "dak_common.cuh"

namespace dak {

constexpr int kKv4Dim = 128;

struct Kv4Cache {
  uint8_t *pool[2];        // device, host
  long long pages[2];
  long long page_bytes;    // all heads of a page
  int slab_bytes;          // one head
  const int32_t *table;
  long long table_stride;
  int max_pages, rows;     // table entries per sequence, sequences
  int kv_heads, page_size, page_log2, ng;
  int *status;
};

__host__ __device__ constexpr int kv4_half_bytes(int page_size, int ng) { return page_size * (64 + 4 * ng); }

__device__ __forceinline__ bool kv4_in_table(const Kv4Cache &c, int seq, int page) {
  return seq >= 0 && seq < c.rows && page >= 0 && page < c.max_pages;
}

// First byte (head 0) of the page that an entry names, or nullptr for an entry
// outside its pool; *tier becomes 0 (device) or 1 (host).
__device__ __forceinline__ uint8_t *kv4_page_of(const Kv4Cache &c, int entry, int *tier) {
  const int t = entry < 0 ? 1 : 0;
  const long long idx = entry < 0 ? -1ll - entry : entry;
  if (idx >= c.pages[t]) return nullptr;
  *tier = t;
  return c.pool[t] + idx * c.page_bytes;
}

// The same for page `page` of sequence `seq`, nullptr outside the table too.
__device__ __forceinline__ uint8_t *kv4_page(const Kv4Cache &c, int seq, int page, int *tier) {
  return kv4_in_table(c, seq, page) ? kv4_page_of(c, c.table[(long long)seq * c.table_stride + page], tier) : nullptr;
}

}  // namespace dak
