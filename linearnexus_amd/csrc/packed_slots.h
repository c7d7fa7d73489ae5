// Slots of a packed batch's blocks, for kernels whose workgroups each take one.
#pragma once
#include "lnx_common.h"

// Blocks of `size` tokens of a packed batch: sequence s takes the slots from first / size + s on, of T / size + nseq in all (a slot or two
// of a sequence may stay empty).  The sequence that owns `slot`: the last one that starts at or before it, found 64 at a time by a
// whole wave.  Always a sequence of the table, and the slots of blocks that exist are within the T / size + nseq, whatever the table holds.
__device__ __forceinline__ int64_t packed_slot(int first, int s, int size) { return (int64_t)(first / size) + s; }
__device__ __forceinline__ int packed_owner(const int32_t* cu, int nseq, int T, int size, int64_t slot) {
  const int lane = threadIdx.x & 63;
  int lo = 0;
  for (int n = nseq; n > 1;) {
    const int step = (int)(((int64_t)n + 63) / 64);
    const int64_t at = (int64_t)lane * step;
    const uint64_t hit = __ballot(at < n && packed_slot(seq_first(cu, lo + (at < n ? (int)at : 0), T), lo + (int)at, size) <= slot);
    const int l = hit ? 63 - __builtin_clzll(hit) : 0;
    lo += l * step;
    n = min(step, n - l * step);
  }
  return __builtin_amdgcn_readfirstlane(lo);
}
