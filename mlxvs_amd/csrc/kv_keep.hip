// The n tokens of each request and kv head that a budget leaves: the first and
// the recent ones, and of the others those of the largest mass, the lowest among
// equal ones, in their order.  A request of at most `above` tokens keeps all: its
// list is empty.
//
// Masses are compared as 32-bit ranks in their order (NaN last), so the list is a
// matter of definition.  A row is a workgroup's: the n-th largest rank 8 bits at a
// time, then the ones above it and the first of those that equal it.
#include <hip/hip_runtime.h>

#include "kv_cache.h"

namespace mlxvs::kern {
namespace {

constexpr uint32_t kAlways = 0xFFFFFFFFu;
constexpr int kThreads = 1024, kWaves = kThreads / 64;

__device__ __forceinline__ int bits(uint64_t x) { return (int)__popcll(x); }

// A mass as a rank: greater masses, greater ranks; -0 and 0 are equal, NaN is 1
// (below minus infinity), 0 stands for no token.
__device__ __forceinline__ uint32_t rank_of(float x) {
  if (x != x) return 1;
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);
  return u >> 31 ? ~u : u | 0x80000000u;
}

__global__ __launch_bounds__(kThreads) void kv_keep_kernel(KvKeepArgs a) {
  __shared__ uint32_t hist[256];
  __shared__ int gt[kWaves], eq[kWaves];
  __shared__ uint32_t found;
  __shared__ int rest;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t r = blockIdx.x / a.heads;
  const int length = (int)min<int64_t>(a.lengths[r], a.slots);
  const float* mass = a.mass + (int64_t)blockIdx.x * a.slots;
  int32_t* out = a.kept + (int64_t)blockIdx.x * a.n;
  if (length <= a.above) {
    for (int i = threadIdx.x; i < a.n; i += kThreads) out[i] = -1;
    return;
  }
  const auto rank = [&](int i) {
    return i < a.first || i >= length - a.recent ? kAlways : rank_of(mass[i]);
  };
  uint32_t cut = 0;
  int left = a.n;
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (threadIdx.x < 256) hist[threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < length; i += kThreads) {
      const uint32_t k = rank(i);
      if (shift == 24 || (k >> (shift + 8)) == (cut >> (shift + 8)))
        atomicAdd(&hist[(k >> shift) & 255], 1u);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int n = 0, b = 255;
      while (b > 0 && n + (int)hist[b] < left) n += (int)hist[b--];
      found = cut | (uint32_t)b << shift;
      rest = left - n;
    }
    __syncthreads();
    cut = found;
    left = rest;
  }
  // each wavefront a stretch of the tokens
  const int per = (length + kThreads - 1) / kThreads * 64;
  const int from = min(length, wave * per), to = min(length, from + per);
  int above = 0, same = 0;
  for (int i = from + lane; i - lane < to; i += 64) {
    const uint32_t k = i < to ? rank(i) : 0;
    above += bits(__ballot(k > cut));
    same += bits(__ballot(k == cut && i < to));
  }
  if (lane == 0) {
    gt[wave] = above;
    eq[wave] = same;
  }
  __syncthreads();
  int at = 0, ties = 0;
  for (int w = 0; w < wave; ++w) {
    at += gt[w] + min(eq[w], max(0, left - ties));
    ties += eq[w];
  }
  const uint64_t below = (uint64_t(1) << lane) - 1;
  for (int i = from + lane; i - lane < to; i += 64) {
    const uint32_t k = i < to ? rank(i) : 0;
    const bool tie = k == cut && i < to;
    const uint64_t tied = __ballot(tie);
    const bool take = k > cut || (tie && ties + bits(tied & below) < left);
    const uint64_t taken = __ballot(take);
    if (take) out[at + bits(taken & below)] = i;
    at += bits(taken);
    ties += bits(tied);
  }
}

}  // namespace

int64_t kv_keep_grid(const KvKeepArgs& a) { return a.requests * a.heads; }

hipError_t launch_kv_keep(const KvKeepArgs& a, hipStream_t s) {
  kv_keep_kernel<<<dim3((unsigned)kv_keep_grid(a)), kThreads, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace mlxvs::kern
