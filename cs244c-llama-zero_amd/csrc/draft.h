// Lookups in a step's tables and in trees of drafted tokens.  What the device
// tables say is not trusted: whatever they hold, the results stay inside.
#pragma once
#include "lz_common.h"

constexpr int kMostNodes = 4096;  // of a tree

// The last b with start[b] <= x, of the B that there are (ascending, start[0] <=
// x): the sequence that entry x belongs to where start are sums before each.
__host__ __device__ __forceinline__ int lz_last_at(const int32_t* start, int B, int x) {
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// A tree's node: its depth (-1: there is no such node) and, where `mask` is not
// null, the words whose bits are itself and its ancestors.  A parent that does
// not come before its child is none, so the way up ends.
__host__ __device__ __forceinline__ int lz_node_depth(const int32_t* parents, int nodes, int node, int32_t* mask, int words) {
  if (mask)
    for (int w = 0; w < words; ++w) mask[w] = 0;
  if (node < 0 || node >= nodes) return -1;
  uint32_t word = 0;
  for (int at = node, w = node >> 5, depth = 0;; ++depth) {
    if (at >> 5 != w) {
      if (mask) mask[w] = (int32_t)word;
      word = 0;
      w = at >> 5;
    }
    word |= 1u << (at & 31);
    const int up = parents[at];
    if (up < 0 || up >= at) {
      if (mask) mask[w] = (int32_t)word;
      return depth;
    }
    at = up;
  }
}
