// Writing new tokens into the paged key-value cache, and the summaries of the
// pages that they complete.
//
// Keys are copied a row at a time, 16 bytes a lane.  Values are transposed
// within a page, through LDS: neighbouring lanes store neighbouring tokens, so
// that a prompt's stores cover whole sectors (16-byte stores of 8 tokens' values
// are slower: 22.7 us, not 20.7, for 4,001 tokens of 5 requests, 4 kv heads of 80
// values).  It moves bytes: 277,688 tokens of 8 x 128 values take 0.59 ms and 0.33
// for the summaries, 3.9 and 1.7 TB/s (the keys are read for their largest, and again
// for the sums); small calls are one launch, 6.8 us.
//
// A page's summary (a page and head): each key value over the largest of the
// page in 127ths, rounded to a whole number; their sums over the page; the sums
// in 127ths of the largest sum: int8 codes, with the scale that makes code x
// scale the mean key.  Sums of whole numbers are the same in every order, so
// codes do not depend on how a page was filled or on how a kernel adds.
#include <hip/hip_runtime.h>

#include "kv_cache.h"
#include "kv_values.h"

namespace mlxvs::kern {
namespace {

// Valid slots name a page of the cache; others are skipped.
__device__ __forceinline__ bool in_cache(const KvCache& c, int64_t slot) {
  return slot >= 0 && (slot >> c.lps) < c.pages;
}
__device__ __forceinline__ bool completes(const KvCache& c, int64_t slot) {
  return in_cache(c, slot) && (slot & (c.page - 1)) == c.page - 1;
}

struct Sums {
  int sum[kKvMaxDim];
  float red[4];
};

// The summary of a page and head by THREADS threads; row(i) is key i's address.
template <bool BF16, int THREADS, typename Row>
__device__ void summarise(const KvCache& c, int64_t at, Sums& s, Row row) {
  const int tid = threadIdx.x, d = c.dim, chunks = d / 8;
  const int rows = THREADS / chunks, x = 8 * (tid % chunks);
  const int i0 = tid < rows * chunks ? tid / chunks : c.page;
  float top = 0.0f, bad = 0.0f;
#pragma unroll 4
  for (int i = i0; i < c.page; i += rows) {
    const uintx4 v = *(const uintx4*)(row(i) + x);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float k = fabsf(value<BF16>(v, j));
      if (!(k < __builtin_inff())) bad = 1.0f;
      top = fmaxf(top, k);
    }
  }
  top = block_max<THREADS>(top, s.red);
  bad = block_max<THREADS>(bad, s.red);
  // nothing to see (or too small to divide by), or a key that is not finite:
  // the block counts as the best, so that what is broken is not left out
  const bool empty = bad != 0.0f || !(top > 1e-30f);
  const float inv = empty ? 0.0f : 127.0f / top;
  for (int i = tid; i < d; i += THREADS) s.sum[i] = 0;
  __syncthreads();
  if (!empty && i0 < c.page) {
    // a thread adds up the keys that it has before the threads meet in LDS
    int part[8] = {};
#pragma unroll 4
    for (int i = i0; i < c.page; i += rows) {
      const uintx4 v = *(const uintx4*)(row(i) + x);
#pragma unroll
      for (int j = 0; j < 8; ++j) part[j] += (int)rintf(value<BF16>(v, j) * inv);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) atomicAdd(&s.sum[x + j], part[j]);
  }
  __syncthreads();
  float peak = 0.0f;
  for (int i = tid; i < d; i += THREADS) peak = fmaxf(peak, (float)abs(s.sum[i]));
  peak = block_max<THREADS>(peak, s.red);
  const float to = peak > 0.0f ? 127.0f / peak : 0.0f;
  for (int i = tid; i < d; i += THREADS)
    c.summaries[at * d + i] = (int8_t)rintf((float)s.sum[i] * to);
  if (tid == 0)
    c.scales[at] = bad != 0.0f ? __builtin_inff()
                   : empty     ? 0.0f
                               : top * (peak / (16129.0f * (float)c.page));
  __syncthreads();
}

// TILE tokens and a head.  FEW: the summaries too, in the same launch: the keys
// of a completed page that this call writes are read where they come from, so
// that no workgroup waits for another's stores (each looks all slots through
// for them, which is why the call's tokens are few).  In one and two launches
// (8 kv heads of 128 values, pages of 64): 256 requests' tokens 9.6 and 16.6 us,
// 1,024 requests' 21.8 and 23.9; one request's 1,024 tokens 9.4 and 9.6, 2,048
// 12.5 and 11.2.
constexpr int kFew = 1024;

template <bool BF16, int TILE, bool FEW>
__global__ __launch_bounds__(256) void kv_append_kernel(KvAppendArgs a) {
  __shared__ uint16_t tile[TILE][kKvMaxDim + 2];
  const int h = (int)(blockIdx.x % a.c.heads);
  const int64_t t0 = (int64_t)(blockIdx.x / a.c.heads) * TILE;
  const int d = a.c.dim, chunks = d / 8;
  const int64_t head = (int64_t)a.c.page * d;
  const int tokens = (int)min<int64_t>(TILE, a.tokens - t0);
  const uint16_t* k = (const uint16_t*)a.k + h * a.k_head;
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
        *(const uintx4*)(k + (t0 + t) * a.k_token + x);
  }
  __syncthreads();
  const int t = threadIdx.x % TILE;
  if (t < tokens) {
    const int64_t slot = a.slots[t0 + t];
    if (in_cache(a.c, slot)) {
      uint16_t* dst = (uint16_t*)a.c.values + ((slot >> a.c.lps) * a.c.heads + h) * head +
                      (slot & (a.c.page - 1));
      for (int i = threadIdx.x / TILE; i < d; i += 256 / TILE) dst[i * a.c.page] = tile[t][i];
    }
  }
  if constexpr (FEW) {
    __shared__ Sums sums;
    __shared__ int from[256];  // a page's keys: the token that writes it now, or -1
    for (int i = 0; i < tokens; ++i) {
      const int64_t slot = a.slots[t0 + i];
      if (!completes(a.c, slot)) continue;
      const int64_t page = slot >> a.c.lps;
      from[threadIdx.x] = -1;
      __syncthreads();
      for (int u = threadIdx.x; u < a.tokens; u += 256) {
        const int64_t other = a.slots[u];
        if (other >= 0 && other >> a.c.lps == page) from[other & (a.c.page - 1)] = u;
      }
      __syncthreads();
      const int64_t at = page * a.c.heads + h;
      const uint16_t* held = (const uint16_t*)a.c.keys + at * head;
      summarise<BF16, 256>(a.c, at, sums, [&](int j) {
        return from[j] >= 0 ? k + from[j] * a.k_token : held + j * d;
      });
    }
  }
}

// Many tokens: the summaries by a launch of their own, a wavefront for `span`
// tokens and a head.
template <bool BF16>
__global__ __launch_bounds__(64) void kv_summaries_kernel(KvAppendArgs a, int span) {
  __shared__ Sums sums;
  const int h = (int)(blockIdx.x % a.c.heads);
  const int64_t t = (int64_t)(blockIdx.x / a.c.heads) * span + threadIdx.x;
  const int64_t slot = (int)threadIdx.x < span && t < a.tokens ? a.slots[t] : -1;
  for (uint64_t todo = __ballot(completes(a.c, slot)); todo; todo &= todo - 1) {
    const int64_t at = (__shfl(slot, __builtin_ctzll(todo)) >> a.c.lps) * a.c.heads + h;
    const uint16_t* held = (const uint16_t*)a.c.keys + at * a.c.page * a.c.dim;
    summarise<BF16, 64>(a.c, at, sums, [&](int j) { return held + j * a.c.dim; });
  }
}

// Whether one launch does it all, and how many tokens its workgroups take then.
// Small tiles: a workgroup's summaries follow one another.  By 4 and 16: 64
// requests' tokens 6.9 and 12.0 us, 512 requests' 12.7 and 17.4 (one request's
// 512 tokens 8.8 and 8.2).
bool few(const KvAppendArgs& a) { return a.tokens <= kFew && a.c.summaries; }
int tile_of(const KvAppendArgs& a) { return few(a) && a.tokens <= 512 ? 4 : 16; }

template <bool BF16, int TILE, bool FEW>
void launch_tile(const KvAppendArgs& a, hipStream_t s) {
  const int64_t grid = (a.tokens + TILE - 1) / TILE * a.c.heads;
  kv_append_kernel<BF16, TILE, FEW><<<dim3((unsigned)grid), 256, 0, s>>>(a);
}

template <bool BF16>
hipError_t launch_append(const KvAppendArgs& a, hipStream_t s) {
  constexpr int kSpan = 16;
  if (few(a)) {
    tile_of(a) == 4 ? launch_tile<BF16, 4, true>(a, s) : launch_tile<BF16, 16, true>(a, s);
    return hipGetLastError();
  }
  launch_tile<BF16, 16, false>(a, s);
  if (hipError_t e = hipGetLastError(); e != hipSuccess || !a.c.summaries) return e;
  const int64_t grid = (a.tokens + kSpan - 1) / kSpan * a.c.heads;
  kv_summaries_kernel<BF16><<<dim3((unsigned)grid), 64, 0, s>>>(a, kSpan);
  return hipGetLastError();
}

}  // namespace

int64_t kv_append_grid(const KvAppendArgs& a) {
  return (a.tokens + tile_of(a) - 1) / tile_of(a) * a.c.heads;
}

hipError_t launch_kv_append(const KvAppendArgs& a, hipStream_t s) {
  return a.c.bf16 ? launch_append<true>(a, s) : launch_append<false>(a, s);
}

}  // namespace mlxvs::kern
