// Copies from global memory straight into LDS (no registers hold the data), and
// the waits and barriers that go with them.
//
// The copies are inline assembly: the compiler knows nothing of their flight, so
// every use waits for them by hand (wait_copies) and then meets the workgroup's
// barrier, which makes all waves' copies visible. They write LDS only, so no
// register is written while one is in flight.
#pragma once
#include "../kernels/moe_numerics.h"

namespace nklds2 {

using nk::u32x4;

__device__ __forceinline__ uint32_t lds_offset(const void* p) {
  return (uint32_t)(size_t)(const __attribute__((address_space(3))) void*)p;
}

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

// 16 bytes per lane, global (r + voff + soff) -> LDS (m0 + 16 * lane). The s_nop
// gives the wait states between a VALU write of the scalar registers or the write
// of m0 and the load, which the compiler does not place around inline assembly; m0
// is put back, as the compiler may keep a value there.
__device__ __forceinline__ void copy16(uint32_t m0, u32x4 r, uint32_t voff, uint32_t soff) {
  uint32_t saved;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 4\n\tbuffer_load_dwordx4 %2, %3, %4 offen lds\n\t"
               "s_mov_b32 m0, %0"
               : "=&s"(saved)
               : "s"(m0), "v"(voff), "s"(r), "s"(soff)
               : "memory");
}

// Two such copies, the second 1 KiB further on both sides (the offset counts for both): a
// 2 KiB tile.
__device__ __forceinline__ void copy_tile(uint32_t m0, u32x4 r, uint32_t voff, uint32_t soff) {
  uint32_t saved;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 4\n\tbuffer_load_dwordx4 %2, %3, %4 offen lds\n\t"
               "buffer_load_dwordx4 %2, %3, %4 offen offset:1024 lds\n\ts_mov_b32 m0, %0"
               : "=&s"(saved)
               : "s"(m0), "v"(voff), "s"(r), "s"(soff)
               : "memory");
}

// 4 bytes per lane -> LDS (m0 + 4 * lane); as copy16.
__device__ __forceinline__ void copy4(uint32_t m0, u32x4 r, uint32_t voff, uint32_t soff) {
  uint32_t saved;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 4\n\tbuffer_load_dword %2, %3, %4 offen lds\n\t"
               "s_mov_b32 m0, %0"
               : "=&s"(saved)
               : "s"(m0), "v"(voff), "s"(r), "s"(soff)
               : "memory");
}

template <uint32_t N>
__device__ __forceinline__ void wait_copies() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}

// Workgroup barrier that drains this wave's LDS traffic but not its copies in flight.
__device__ __forceinline__ void barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

}  // namespace nklds2
