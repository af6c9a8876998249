// What the paged cache's kernels share of values and workgroups.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mlxvs::kern {

typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));

// A binary16 or bfloat16 value.
template <bool BF16>
__device__ __forceinline__ float value(uint16_t x) {
  if constexpr (BF16) return __builtin_bit_cast(float, (uint32_t)x << 16);
  else return (float)__builtin_bit_cast(_Float16, x);
}

// The j-th of 8 of them.
template <bool BF16>
__device__ __forceinline__ float value(const uintx4& v, int j) {
  return value<BF16>((uint16_t)(v[j / 2] >> (16 * (j & 1))));
}

// The largest x of a wavefront, of a workgroup of THREADS (shared: a place for
// each of its wavefronts).
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int i = 32; i >= 1; i >>= 1) x = fmaxf(x, __shfl_xor(x, i));
  return x;
}
template <int THREADS>
__device__ __forceinline__ float block_max(float x, float* shared) {
  x = wave_max(x);
  if constexpr (THREADS == 64) return x;
  if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = x;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < THREADS / 64; ++i) x = fmaxf(x, shared[i]);
  __syncthreads();
  return x;
}

}  // namespace mlxvs::kern
