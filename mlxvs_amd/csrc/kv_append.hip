// Writing new tokens into the paged key-value cache, and the summaries of the
// pages that they complete.
//
// Keys are copied a row at a time, 16 bytes a lane.  Values are transposed
// within a page, through LDS: neighbouring lanes store neighbouring tokens, so
// that a prompt's stores cover whole sectors.
//
// A page's summary (a page and head): each key value over the largest of the
// page in 127ths, rounded to a whole number; their sums over the page; the sums
// in 127ths of the largest sum: int8 codes, with the scale that makes code x
// scale the mean key.  Sums of whole numbers are the same in every order, so
// codes do not depend on how a page was filled or on how a kernel adds.
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include "kv_cache.h"

namespace mlxvs::kern {
namespace {

typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 16;  // tokens of a workgroup

// Valid slots name a page of the cache; others are skipped.
__device__ __forceinline__ bool in_cache(const KvCache& c, int64_t slot) {
  return slot >= 0 && (slot >> c.lps) < c.pages;
}

__global__ __launch_bounds__(256) void kv_append_kernel(KvAppendArgs a) {
  __shared__ uint16_t tile[kTile][kKvMaxDim + 2];
  const int h = (int)(blockIdx.x % a.c.heads);
  const int64_t t0 = (int64_t)(blockIdx.x / a.c.heads) * kTile;
  const int d = a.c.dim, chunks = d / 8;
  const int64_t head = (int64_t)a.c.page * d;
  const int tokens = (int)min<int64_t>(kTile, a.tokens - t0);
  for (int i = threadIdx.x; i < tokens * chunks; i += 256) {
    const int t = i / chunks, x = 8 * (i % chunks);
    const int64_t slot = a.slots[t0 + t];
    const uintx4 v = *(const uintx4*)((const uint16_t*)a.v + (t0 + t) * a.v_token +
                                      h * a.v_head + x);
#pragma unroll
    for (int j = 0; j < 4; ++j) *(uint32_t*)&tile[t][x + 2 * j] = v[j];
    if (!in_cache(a.c, slot)) continue;
    const int64_t page = slot >> a.c.lps;
    const int off = (int)(slot & (a.c.page - 1));
    *(uintx4*)((uint16_t*)a.c.keys + (page * a.c.heads + h) * head + off * d + x) =
        *(const uintx4*)((const uint16_t*)a.k + (t0 + t) * a.k_token + h * a.k_head + x);
  }
  __syncthreads();
  const int t = threadIdx.x % kTile;
  if (t >= tokens) return;
  const int64_t slot = a.slots[t0 + t];
  if (!in_cache(a.c, slot)) return;
  uint16_t* dst = (uint16_t*)a.c.values + ((slot >> a.c.lps) * a.c.heads + h) * head +
                  (slot & (a.c.page - 1));
  for (int i = threadIdx.x / kTile; i < d; i += 256 / kTile) dst[i * a.c.page] = tile[t][i];
}

template <bool BF16>
__device__ __forceinline__ float value(uint16_t x) {
  if constexpr (BF16) return __builtin_bit_cast(float, (uint32_t)x << 16);
  else return (float)__builtin_bit_cast(_Float16, x);
}

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int i = 32; i >= 1; i >>= 1) x = fmaxf(x, __shfl_xor(x, i));
  return x;
}

// One page and head, by one wavefront.
template <bool BF16>
__device__ void summarise(const KvCache& c, int64_t page, int h, int* sums) {
  const int lane = threadIdx.x, d = c.dim, chunks = d / 8;
  const int64_t at = page * c.heads + h;
  const uint16_t* keys = (const uint16_t*)c.keys + at * c.page * d;
  float top = 0.0f;
  bool finite = true;
  for (int i = lane; i < c.page * chunks; i += 64) {
    const uintx4 v = *(const uintx4*)(keys + 8 * i);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float x = fabsf(value<BF16>((uint16_t)(v[j / 2] >> (16 * (j & 1)))));
      finite &= x < __builtin_inff();
      top = fmaxf(top, x);
    }
  }
  top = wave_max(top);
  finite = __all(finite);
  // nothing to see (or too small to divide by), or a key that is not finite:
  // the block counts as the best, so that what is broken is not left out
  const bool empty = !finite || !(top > 1e-30f);
  const float inv = empty ? 0.0f : 127.0f / top;
  for (int i = lane; i < d; i += 64) sums[i] = 0;
  __syncthreads();
  if (!empty) {
    // lanes of one 8-value chunk add what they have before they meet in LDS
    const int rows = 64 / chunks, x = lane % chunks;
    if (lane < rows * chunks) {
      int part[8] = {};
      for (int i = lane / chunks; i < c.page; i += rows) {
        const uintx4 v = *(const uintx4*)(keys + i * d + 8 * x);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          part[j] += (int)rintf(value<BF16>((uint16_t)(v[j / 2] >> (16 * (j & 1)))) * inv);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) atomicAdd(&sums[8 * x + j], part[j]);
    }
  }
  __syncthreads();
  float peak = 0.0f;
  for (int i = lane; i < d; i += 64) peak = fmaxf(peak, (float)abs(sums[i]));
  peak = wave_max(peak);
  const float to = peak > 0.0f ? 127.0f / peak : 0.0f;
  for (int i = lane; i < d; i += 64) c.summaries[at * d + i] = (int8_t)rintf((float)sums[i] * to);
  if (lane == 0)
    c.scales[at] = !finite ? __builtin_inff()
                           : empty ? 0.0f : top * (peak / (16129.0f * (float)c.page));
  __syncthreads();
}

// A wavefront for `span` tokens and a head.
template <bool BF16>
__global__ __launch_bounds__(64) void kv_summaries_kernel(KvAppendArgs a, int span) {
  __shared__ int sums[kKvMaxDim];
  const int h = (int)(blockIdx.x % a.c.heads);
  const int64_t t0 = (int64_t)(blockIdx.x / a.c.heads) * span;
  const int64_t t = t0 + threadIdx.x;
  const int64_t slot = (int)threadIdx.x < span && t < a.tokens ? a.slots[t] : -1;
  const bool last = in_cache(a.c, slot) && (slot & (a.c.page - 1)) == a.c.page - 1;
  for (uint64_t todo = __ballot(last); todo; todo &= todo - 1) {
    const int from = __builtin_ctzll(todo);
    summarise<BF16>(a.c, __shfl(slot, from) >> a.c.lps, h, sums);
  }
}

}  // namespace

hipError_t launch_kv_append(const KvAppendArgs& a, hipStream_t s) {
  const int64_t grid = (a.tokens + kTile - 1) / kTile * a.c.heads;
  kv_append_kernel<<<dim3((unsigned)grid), 256, 0, s>>>(a);
  return hipGetLastError();
}

hipError_t launch_kv_summaries(const KvAppendArgs& a, hipStream_t s) {
  const int span = a.tokens > 1024 ? 16 : 1;
  const int64_t grid = (a.tokens + span - 1) / span * a.c.heads;
  if (a.c.bf16) kv_summaries_kernel<true><<<dim3((unsigned)grid), 64, 0, s>>>(a, span);
  else kv_summaries_kernel<false><<<dim3((unsigned)grid), 64, 0, s>>>(a, span);
  return hipGetLastError();
}

}  // namespace mlxvs::kern
