// What the linear layer's tiles add to the copies into LDS: a descriptor in scalar
// registers, and a whole tile per copy.
#pragma once
#include "../kernels/lds_copy.h"

namespace nklds2 {

using nk::u32x4;
using nklds::barrier;
using nklds::copy16;
using nklds::copy4;
using nklds::lds_offset;
using nklds::wait_copies;

// Raw buffer descriptor over `bytes` bytes from base; reads past them give zeros
// without touching memory.
__device__ __forceinline__ u32x4 rsrc(const void* base, uint32_t bytes) {
  const uint64_t a = (uint64_t)base;
  u32x4 r;
  r.x = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a);
  r.y = (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(a >> 32) & 0xffffu));
  r.z = (uint32_t)__builtin_amdgcn_readfirstlane((int)bytes);
  r.w = 0x00020000u;
  return r;
}

// Two of copy16, the second 1 KiB further on both sides (the offset counts for both): a
// 2 KiB tile.
__device__ __forceinline__ void copy_tile(uint32_t m0, u32x4 r, uint32_t voff, uint32_t soff) {
  uint32_t saved;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 4\n\tbuffer_load_dwordx4 %2, %3, %4 offen lds\n\t"
               "buffer_load_dwordx4 %2, %3, %4 offen offset:1024 lds\n\ts_mov_b32 m0, %0"
               : "=&s"(saved)
               : "s"(m0), "v"(voff), "s"(r), "s"(soff)
               : "memory");
}

}  // namespace nklds2
