// The summary of a page and head of the paged cache.
//
// Each key value over the largest of the page in 127ths, rounded to a whole
// number; their sums over the page; the sums in 127ths of the largest sum: int8
// codes, with the scale that makes code x scale the mean key.  Sums of whole
// numbers are the same in every order, so codes do not depend on how a page was
// filled or on how a kernel adds.
#pragma once

#include <hip/hip_runtime.h>

#include "kv_cache.h"
#include "kv_values.h"

namespace mlxvs::kern {

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

}  // namespace mlxvs::kern
