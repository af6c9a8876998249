// Staging rows in LDS for the MFMA kernels: direct loads and the waits around
// them.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mlxvs::kern {

// Buffer loads of 16 / 4 bytes per lane straight into LDS: lane l writes at
// lds + 16 l (4 l); lds is wavefront-uniform; out-of-range lanes write
// zeros.  (The builtin exists only for the device target.)
__device__ __forceinline__ void load16_to_lds(__amdgpu_buffer_rsrc_t r, void* lds, uint32_t voff) {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 16,
                                           voff, 0, 0, 0);
#else
  (void)r, (void)lds, (void)voff;
#endif
}
__device__ __forceinline__ void load4_to_lds(__amdgpu_buffer_rsrc_t r, void* lds, uint32_t voff) {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 4,
                                           voff, 0, 0, 0);
#else
  (void)r, (void)lds, (void)voff;
#endif
}

// 16 bytes a lane from `from` to lds + 16 lane.
__device__ __forceinline__ void copy16_to_lds(const void* from, void* lds) {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                   (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
#endif
}

// A place in LDS as the instructions take it, and 16 bytes from one.
__device__ __forceinline__ uint32_t lds_address(const void* lds) {
#if defined(__HIP_DEVICE_COMPILE__)
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)lds;
#else
  return 0;
#endif
}
__device__ __forceinline__ auto lds_read16(uint32_t at) {
  typedef uint32_t uintx4_t __attribute__((ext_vector_type(4)));
#if defined(__HIP_DEVICE_COMPILE__)
  return *(const __attribute__((address_space(3))) uintx4_t*)(uintptr_t)at;
#else
  return uintx4_t{};
#endif
}

template <typename T>
__device__ __forceinline__ T lds_read4(uint32_t at) {
  static_assert(sizeof(T) == 4);
#if defined(__HIP_DEVICE_COMPILE__)
  return *(const __attribute__((address_space(3))) T*)(uintptr_t)at;
#else
  return T{};
#endif
}

// Direct loads of 16 or 4 bytes a lane for tiles that are several loads ahead.  The
// compiler waits for all loads like those above before it reads any LDS that one of
// them may have written, and takes every buffer for such; of these it knows
// nothing: whoever reads what they bring waits for them (staged_barrier).  They
// return nothing to registers.  The place in LDS is the wavefront's.  (m0 is named as
// written, of which the compiler warns, since it has uses for it itself.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void stream16_to_lds(const void* from, uint32_t lds) {
#if defined(__HIP_DEVICE_COMPILE__)
  const int to = __builtin_amdgcn_readfirstlane((int)lds);
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
               ::"v"(from), "s"(to) : "memory", "m0");
#endif
}
__device__ __forceinline__ void stream4_to_lds(const void* from, uint32_t lds) {
#if defined(__HIP_DEVICE_COMPILE__)
  const int to = __builtin_amdgcn_readfirstlane((int)lds);
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off"
               ::"v"(from), "s"(to) : "memory", "m0");
#endif
}
#pragma clang diagnostic pop

// A workgroup barrier once all but the latest LEFT of this wavefront's loads are
// done, for buffers that stream*_to_lds fill.
template <int LEFT>
__device__ __forceinline__ void staged_barrier() {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LEFT) : "memory");
  __builtin_amdgcn_sched_barrier(0);
#endif
}

// A workgroup barrier after this wavefront's outstanding vector-memory
// operations -- its LDS-direct loads among them -- have completed: an LDS
// buffer that every wavefront fills with LDS-direct loads is whole once all
// have passed it.  (The barrier's own workgroup-scope fence does not wait
// for loads, so the wait is explicit.)
__device__ __forceinline__ void dma_barrier() {
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0), no other counter
  __syncthreads();
}

// Wait states between a barrier and the first read of MFMA results issued
// before it.  The compiler's MFMA-to-VALU dependency count includes the
// barrier and the wait in front of it, which need not take a cycle (a
// wavefront that arrives last passes both at once): reading the last
// accumulator registers first, at the count it derived, gave stale values
// now and then (lists that lost a candidate, measured on the GPU: gone with
// 8 more wait states, not with 1).  Twenty-four, fenced so that nothing is
// scheduled across them: more than the longest MFMA here needs (16 passes
// + 2) whether or not the compiler counts them towards its own.
__device__ __forceinline__ void mfma_settle() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7");
  __builtin_amdgcn_sched_barrier(0);
}

}  // namespace mlxvs::kern
