// lds_copy.h -- copies from global memory straight into LDS that the compiler does not
// wait for by itself, and the waits for them (linear.hip, the MXFP4 products).
#pragma once

#include "exq_internal.h"

namespace exq {
namespace lin {

// 16 bytes per lane from buffer `r` at byte offset voff + soff into LDS at
// lds + 16 * lane; `lds` and `soff` are wave-uniform.  A voff past the resource
// writes zeros and reads nothing.  Inline asm (it has no output register), as the
// compiler puts a wait for all copies in flight before the next LDS read after its
// own builtin, which ends the overlap that the stages are for; every copy here is
// waited for by count (wait_vm) and, across waves, by a barrier.  The LDS address is
// an operand in m0, so the compiler knows that m0 changes here.
typedef void __attribute__((address_space(3)))* lptr_t;
__device__ __forceinline__ uint32_t lds_offset(const unsigned char* p) {
  return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lptr_t)p);
}
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t r, uint32_t lds, int voff, int soff) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"{m0}"(lds), "v"(voff),
               "s"(r), "s"(soff)
               : "memory");
#endif
}
// The same for four bytes a lane from anywhere.
__device__ __forceinline__ void touch(const uint16_t* p, uint32_t lds) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_nop 0\n\tglobal_load_lds_dword %1, off" ::"{m0}"(lds), "v"(p) : "memory");
#endif
}
constexpr int kOob = 0x7ffffff0;          // a voff past every resource
constexpr int64_t kSpan = 0x7fffff00;     // bytes that one resource covers at most
__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const uint16_t* base) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(base), (short)0, (int)kSpan,
                                           0x00020000);
}
// LDS written by a copy is ordered only by the vmcnt wait, which the compiler does
// not see as a dependency: volatile asm that no memory access moves across.
template <int N>
__device__ __forceinline__ void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

}  // namespace lin
}  // namespace exq
