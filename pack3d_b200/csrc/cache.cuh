// Pages of keys and values: where a token of a sequence lies, shared by the cache's kernels and the attention over it.
#pragma once

#include "common.cuh"

namespace p3d {
namespace cache {

constexpr unsigned kErrPage = 64u;   // p3d_device_errors: a page outside the cache

// Offsets of packed sequences: the first counts as 0, and none lies past `rows`.
__device__ __forceinline__ int offset_at(const int32_t *offsets, int b, int rows) {
  return b == 0 ? 0 : min(max(offsets[b], 0), rows);
}

// The last sequence that begins at or before row t; rows of no sequence lie behind the end of the one found.
__device__ __forceinline__ int sequence_of(const int32_t *offsets, int sequences, int rows, int t) {
  int lo = 0, hi = sequences;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (offset_at(offsets, mid, rows) <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

// The page of place `at` (a token's number in its sequence) and the row in it; -1 where the table has none. Places are below 2^31.
struct Place {
  int page, row;
};
__device__ __forceinline__ Place place_of(const p3d_cache &c, int b, int64_t at) {
  Place p = {-1, 0};
  if (at < 0 || at >= (int64_t)c.table_width * c.page_size) return p;
  const unsigned i = (unsigned)at / (unsigned)c.page_size;
  p.row = (int)((unsigned)at - i * (unsigned)c.page_size);
  const int page = c.table[b * c.table_stride + i];
  p.page = page >= 0 && page < c.pages ? page : -1;
  return p;
}

int check(const p3d_cache *c, const char *what);   // cache.cu: everything but the data pointers' use

}  // namespace cache
}  // namespace p3d
