// Trees of drafted tokens, as the kernels around speculative decoding read them: the nodes of all trees lie packed, tree b holds
// rows [cu[b], cu[b + 1]). Node 0 of a tree is its root, the last token of the request; parents[row] of any other node is the number
// (within its tree) of an EARLIER node. A node whose parent is anything else belongs to no tree, and neither do the nodes below it:
// such a node sees nothing and is never accepted. With that rule every walk towards the root goes to smaller numbers and ends.
#pragma once

#include "common.cuh"

namespace sb {

constexpr int TREE_MAX = 128;  // nodes of a tree
constexpr long TREE_MAX_KEYS = 0x7fffff00l;  // keys that a request can have: nodes behind them, and the rest of their tile, stay within an int

// Tree of packed row t: the largest b with cu[b] <= t, given cu[0] <= t < cu[B].
__device__ __forceinline__ int tree_of_row(const int* __restrict__ cu, int B, int t) {
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Set of node i and the nodes above it (bit j of word j / 32); empty where the way up does not end at the root.
template <typename Parents>
__device__ __forceinline__ void tree_way_up(const Parents& parent, int i, uint32_t (&set)[4]) {
#pragma unroll
  for (int w = 0; w < 4; ++w) set[w] = 0;
  while (true) {
#pragma unroll
    for (int w = 0; w < 4; ++w)
      if (i >> 5 == w) set[w] |= 1u << (i & 31);
    if (i == 0) return;
    const int up = parent(i);
    if (up < 0 || up >= i) break;
    i = up;
  }
#pragma unroll
  for (int w = 0; w < 4; ++w) set[w] = 0;
}

}  // namespace sb
