// Requests from memory straight into LDS, and their waits (kernels_layered.hip,
// kernels_experts.hip).
#pragma once

#include <hip/hip_runtime.h>

namespace ponni_hip {

// One 16- or 4-byte request per lane into LDS at lds + size * lane (lds
// uniform), as inline asm so that the compiler's wait insertion does not
// wait for every request before each LDS read; the waits below order them
// (the s_nop is the wait state between the write of M0 and its use).
__device__ inline void dma16(void const* g, unsigned lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(g), "{m0}"(lds) : "memory");
}
// The same at a uniform address and a 32-bit offset per lane.  (Five wait states:
// those between a VALU write of a scalar register, as v_readfirstlane's of the
// address, and a memory instruction's read of it, which the hardware does not check.)
__device__ inline void dma16(void const* base, unsigned offset, unsigned lds) {
  asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "{m0}"(lds) : "memory");
}
__device__ inline void dma4(void const* g, unsigned lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(g), "{m0}"(lds) : "memory");
}
// At most N requests of this wave outstanding, and its LDS accesses done.
template <int N>
__device__ inline void wait_requests() {
  static_assert(N >= 0 && N < 64, "vmcnt field");
  __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | (N >> 4) << 14);
}
// This wave's LDS reads have their data.
__device__ inline void wait_lds() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xc07f);
}
__device__ inline void workgroup_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

}  // namespace ponni_hip
