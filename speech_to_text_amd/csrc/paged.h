// Shared by the kernels that deal with drafted token trees.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

// Path of each node of one tree as a 64-bit set, by pointer jumping: after s rounds a node's set holds
// its nearest 2^s ancestors.  Lane l computes node l; parents outside [0, own index) are roots, `parents`
// null is a chain.  `nodes` in 1 .. 64; no branch, so that no register is spilled under a partial mask.
__device__ __forceinline__ unsigned long long tree_path(const int32_t* parents, int row0, int nodes, int lane) {
  const int at = lane < nodes ? lane : nodes - 1;
  int up = parents ? parents[row0 + at] : lane - 1;
  up = lane < nodes && up < lane ? up : -1;
  unsigned long long seen = 1ull << lane;
#pragma unroll
  for (int s = 0; s < 6; ++s) {
    const int src = up < 0 ? lane : up;
    const unsigned long long more = __shfl(seen, src, 64);
    const int next = __shfl(up, src, 64);
    seen |= up >= 0 ? more : 0ull;
    up = up >= 0 ? next : up;
  }
  return seen;
}
