// Direct-to-LDS loads (gfx950: 16 bytes per lane) and their waits.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace qe {
namespace {

// One direct-to-LDS load of a wave: lane l's 16 bytes at `src` go to LDS byte address lds + 16 l.
// The compiler does not count it: a reader waits with wait_dma first. (No output registers.)
__device__ __forceinline__ void dma16(uint32_t lds, const void* src) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(lds), "v"(src) : "memory", "m0");
}
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return uint32_t(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) void*)p));
}
template <int N>
__device__ __forceinline__ void wait_dma() {  // all but the wave's last N vector memory operations are done
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}
__device__ __forceinline__ void wait_lds() {  // the wave's LDS reads have returned
  asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
}

}  // namespace
}  // namespace qe
