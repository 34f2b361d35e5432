// The 8-bit key/value cache: pages of E4M3 codes with one E8M0 scale per page, head and side.
//
//   K codes [pages, kv_heads, page, D]     a page and head: token rows, 1 D page byte run
//   V codes [pages, kv_heads, D, page]     transposed, so that the keys of a channel are
//                                          contiguous: the A operand of Vᵀ Pᵀ as it lies in memory
//   scales  [pages, kv_heads] bytes e + 127 of each side; a code stands for E4M3 * 2^e
//
// page is a power of two from 16 to 256. The tokens of sequence i lie in the pages that row i of
// the table names, in order. Page ids and lengths come from device memory: every kernel checks
// them against the pool and the table and raises *faults instead of following a bad one.
#pragma once

#include "mxfp8_common.h"

namespace vdn {

struct KvCache {
  uint8_t* k;
  uint8_t* ks;
  uint8_t* v;
  uint8_t* vs;
  int* faults;
  int pages, kv_heads, log_page;
};

// Scales start at 2^-100: 2^e and every code's value then are normal in fp32 and bf16. Below that a
// page's values are rounded as E4M3 numbers times 2^-100: by 2^-4 relative, under 2^-106 by 2^-110.
constexpr uint32_t kLeastScaleByte = 27;

// Scale byte of a block from its largest finite magnitude: the least e with amax <= 448 * 2^e.
__device__ __forceinline__ uint32_t cache_scale_byte(float amax) {
  float inv;
  const uint32_t byte = e8m0_from_amax(amax, &inv);
  return byte < kLeastScaleByte ? kLeastScaleByte : byte;
}

// Page id of position `index` of a table row, or -1 (and *faults = 1) if the table or the pool
// does not have it.
__device__ __forceinline__ int cache_page(const KvCache& c, const int* __restrict__ row, int index,
                                          int width) {
  const int id = index >= 0 && index < width ? row[index] : -1;
  if (id >= 0 && id < c.pages) return id;
  *c.faults = 1;
  return -1;
}

// Host: the arguments that every cache entry point shares.
inline bool cache_geometry_ok(const KvCache& c, int page, int head_dim) {
  return c.pages > 0 && c.kv_heads > 0 && page >= 16 && page <= 256 && (page & (page - 1)) == 0 &&
         (head_dim == 64 || head_dim == 128 || head_dim == 256);
}

}  // namespace vdn
