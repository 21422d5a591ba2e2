// Copies from global memory straight into LDS (no registers hold the data), and
// the waits and barriers that go with them.
//
// The copies are inline assembly: the compiler knows nothing of their flight, so
// every use waits for them by hand (wait_copies) and then meets the workgroup's
// barrier, which makes all waves' copies visible. They write LDS only, so no
// register is written while one is in flight.
#pragma once
#include "moe_numerics.h"

namespace nklds {

using nk::u32x4;

__device__ __forceinline__ uint32_t lds_offset(const void* p) {
  return (uint32_t)(size_t)(const __attribute__((address_space(3))) void*)p;
}

// 16 bytes per lane, global (rsrc + voff + soff) -> LDS (m0 + 16 * lane).
// Offsets at or past num_records read as zeros without a memory access.
// The compiler's hazard recognizer does not look inside inline assembly, so
// the s_nop 4 supplies the five wait states a vector-memory instruction needs
// after a VALU write (v_readfirstlane, v_readlane, carry outputs) of an SGPR
// it reads (resource, offset), which also covers the M0 write before an
// LDS-destination load. The compiler treats m0 as a reserved register and
// does not honour it in a clobber list, so the copy saves m0 and puts it back
// (the LDS address is taken from m0 when the load issues): any value the
// compiler keeps in m0 survives the copy.
__device__ __forceinline__ void copy16(uint32_t m0, u32x4 r, uint32_t voff, uint32_t soff) {
  uint32_t saved;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 4\n\tbuffer_load_dwordx4 %2, %3, %4 offen lds\n\t"
               "s_mov_b32 m0, %0"
               : "=&s"(saved)
               : "s"(m0), "v"(voff), "s"(r), "s"(soff)
               : "memory");
}

// 4 bytes per lane, global (rsrc + voff + soff) -> LDS (m0 + 4 * lane); as copy16.
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

// Barrier for LDS hand-off: waits for this wave's LDS traffic, not for its
// copies in flight (a full __syncthreads would drain those).
__device__ __forceinline__ void barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

}  // namespace nklds
