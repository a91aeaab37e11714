// Copies HBM -> LDS without register staging, and the wait for them; for the
// tiled GEMM kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace pa {

// A wavefront's copy HBM -> LDS of 16 bytes per lane: lane l's bytes come
// from base + off (off per lane) and land at LDS address lds + 16 l.  Written
// out in assembly: with the builtin the compiler cannot tell that the operand
// reads which follow use another LDS buffer, and makes them wait for the copy
// (vmcnt(0) right after every copy).  The kernel orders copies and reads
// itself (wait_copies and a barrier at the top of every step).  A load to LDS
// needs one wait state after the write of m0, which the compiler does not add
// inside assembly: the s_nop.
#pragma clang diagnostic ignored "-Winline-asm"  // m0 as a clobber
__device__ inline void lds_copy16(const uint8_t* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               :
               : "v"(off), "s"(base), "s"(lds)
               : "memory", "m0");
}
__device__ inline void lds_copy16(const uint8_t* base, uint64_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
               :
               : "v"(base + off), "s"(lds)
               : "memory", "m0");
}
// The same of 4 bytes per lane, to lds + 4 l.
__device__ inline void lds_copy4(const uint8_t* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1"
               :
               : "v"(off), "s"(base), "s"(lds)
               : "memory", "m0");
}
// Waits until at most N of this wavefront's copies are in flight and its LDS
// reads and writes are done.
template <int N>
__device__ inline void wait_copies() {
  static_assert(N <= 63, "vmcnt range");
  __builtin_amdgcn_s_waitcnt(0x0070 | (N & 0xF) | ((N >> 4) << 14));
}
// Waits until at most N of this wavefront's loads and copies are in flight (no
// wait for its LDS accesses).
template <int N>
__device__ inline void wait_vm() {
  static_assert(N <= 63, "vmcnt range");
  __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 0xF) | ((N >> 4) << 14));
}

}  // namespace pa
