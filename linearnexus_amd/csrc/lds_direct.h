// Loads that go straight to LDS from a wave's base address (those from addresses of each lane are in mma_tiles.h).
#pragma once
#include "mma_tiles.h"

// 16 bytes a lane from `base` + off bytes straight to LDS, lane l at dst + 16 l; the base is the wave's, so a tile's loads cost no
// vector arithmetic
__device__ __forceinline__ void dma16_at(const void* base, unsigned off, unsigned dst) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(__builtin_amdgcn_readfirstlane(dst)) : "memory", "m0");
}
