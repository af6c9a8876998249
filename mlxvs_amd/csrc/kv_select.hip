// The best blocks of a paged cache for every new token: a cheap score of each
// block's summary, and the n best by it.
//
// The query of a (token, kv head): each value of its group's heads over the
// largest of all of them in 127ths, rounded to whole numbers; their sums over
// the heads; the sums in 127ths of the largest.  A block's score is the exact
// int8 dot product of that with the summary's codes, in float32 (below 2^24:
// exact), times the summary's scale.  So the order of the blocks is a matter of
// definition and not of rounding: every split, tile or kernel lists the same
// blocks.  Candidates are the complete blocks before the token's own; its own,
// the latest and the first ones are always taken.
//
// Ranks are 32-bit keys in the scores' order: 0 for no candidate, all ones for
// a block that is always taken.
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>

#include "kv_cache.h"

namespace mlxvs::kern {
namespace {

typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx2 __attribute__((ext_vector_type(2)));

constexpr uint32_t kAlways = 0xFFFFFFFFu;
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kLdsCols = 8192;  // ranks of a row that stay in LDS (32 KB)

template <bool BF16>
__device__ __forceinline__ float value(uint16_t x) {
  if constexpr (BF16) return __builtin_bit_cast(float, (uint32_t)x << 16);
  else return (float)__builtin_bit_cast(_Float16, x);
}

__device__ __forceinline__ uint32_t rank_of(int dot, float scale) {
  // a summary that is not finite ranks first (a broken block is not left out)
  float x = scale < __builtin_inff() ? (float)dot * scale : FLT_MAX;
  x = fminf(fmaxf(x, -FLT_MAX), FLT_MAX) + 0.0f;  // (-0 and 0 are equal)
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  return u >> 31 ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float block_max(float x, float* shared) {
#pragma unroll
  for (int i = 32; i >= 1; i >>= 1) x = fmaxf(x, __shfl_xor(x, i));
  if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = x;
  __syncthreads();
  float y = shared[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) y = fmaxf(y, shared[i]);
  __syncthreads();
  return y;
}

// The codes of a (token, head)'s query, zeros past dim.  A query that holds
// nothing, or a value that is not finite, has codes 0.
template <bool BF16>
__device__ void query_codes(const KvSelectArgs& a, int64_t t, int h, int8_t* codes,
                            float* shared) {
  const int d = threadIdx.x, g = a.q.group;
  const uint16_t* q = (const uint16_t*)a.q.q + t * a.q.q_token + (int64_t)h * g * a.q.q_head + d;
  float top = 0.0f, bad = 0.0f;
  if (d < a.c.dim)
    for (int i = 0; i < g; ++i) {
      const float x = fabsf(value<BF16>(q[i * a.q.q_head]));
      if (!(x < __builtin_inff())) bad = 1.0f;
      top = fmaxf(top, x);
    }
  top = block_max(top, shared);
  bad = block_max(bad, shared);
  const float inv = bad == 0.0f && top > 1e-30f ? 127.0f / top : 0.0f;
  int sum = 0;
  if (d < a.c.dim && inv != 0.0f)
    for (int i = 0; i < g; ++i) sum += (int)rintf(value<BF16>(q[i * a.q.q_head]) * inv);
  const float peak = block_max((float)abs(sum), shared);
  const float to = peak > 0.0f ? 127.0f / peak : 0.0f;
  codes[d] = (int8_t)rintf((float)sum * to);
  __syncthreads();
}

// Ranks of the columns [c0, c1) of a row into ranks[0 ..], lanes of a page's
// group adding up their parts of its dot product.  CH: bytes a lane loads.
template <int CH>
__device__ void rank_columns(const KvSelectArgs& a, int h, int r, int own, int c0, int c1,
                             const int8_t* codes, uint32_t* ranks) {
  const int d = a.c.dim, chunks = d / CH;
  int lanes = 1;
  while (lanes < chunks) lanes *= 2;
  const int at = threadIdx.x % lanes, per = kThreads / lanes;
  uint32_t q[CH / 4];
#pragma unroll
  for (int i = 0; i < CH / 4; ++i) q[i] = at < chunks ? *(const uint32_t*)(codes + CH * at + 4 * i) : 0;
  for (int j0 = c0; j0 < c1; j0 += per) {
    const int j = j0 + (int)threadIdx.x / lanes;
    const int p = j < c1 ? a.q.table[(int64_t)r * a.q.table_stride + j] : -1;
    const bool there = p >= 0 && p < a.c.pages;
    const int64_t row = ((int64_t)p * a.c.heads + h);
    int dot = 0;
    if (there && at < chunks) {
      const int8_t* m = a.c.summaries + row * d + CH * at;
      if constexpr (CH == 16) {
        const uintx4 v = *(const uintx4*)m;
#pragma unroll
        for (int i = 0; i < 4; ++i) dot = __builtin_amdgcn_sdot4((int)v[i], (int)q[i], dot, false);
      } else {
        const uintx2 v = *(const uintx2*)m;
#pragma unroll
        for (int i = 0; i < 2; ++i) dot = __builtin_amdgcn_sdot4((int)v[i], (int)q[i], dot, false);
      }
    }
    for (int x = 1; x < lanes; x *= 2) dot += __shfl_xor(dot, x);
    if (at == 0 && j < c1) {
      uint32_t k = 0;
      if (there) k = j < a.first || j > own - a.last ? kAlways : rank_of(dot, a.c.scales[row]);
      ranks[j - c0] = k;
    }
  }
}

struct Select {
  uint32_t hist[256];
  int gt[kWaves], eq[kWaves];
  uint32_t prefix;
  int left;
};

// The n largest of ranks[0 .. count), the lowest columns among equal ones,
// ascending by column into out, -1 after.
__device__ void take_best(const uint32_t* ranks, int count, int n, int32_t* out, Select& s) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // the n-th largest rank, 8 bits at a time
  uint32_t prefix = 0;
  int left = n;
  if (count > n) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      s.hist[threadIdx.x] = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < count; i += kThreads) {
        const uint32_t k = ranks[i];
        if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8)))
          atomicAdd(&s.hist[(k >> shift) & 255], 1u);
      }
      __syncthreads();
      if (wave == 0) {
        // lane l: bins 4 l .. 4 l + 3, counted from the top
        int c[4], sum = 0;
#pragma unroll
        for (int i = 3; i >= 0; --i) c[i] = sum += (int)s.hist[4 * lane + i];
        int above = sum;
#pragma unroll
        for (int x = 1; x < 64; x *= 2) {
          const int y = __shfl_down(above, x);
          if (lane + x < 64) above += y;
        }
        above -= sum;  // in the bins of the lanes past this one
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int upto = above + c[i], before = i < 3 ? above + c[i + 1] : above;
          if (before < left && upto >= left) {
            s.prefix = prefix | (uint32_t)(4 * lane + i) << shift;
            s.left = left - before;
          }
        }
      }
      __syncthreads();
      prefix = s.prefix;
      left = s.left;
    }
  }
  // each wavefront a stretch of the columns: those above the n-th, and the
  // first `left` that equal it (all that are candidates, if they are few)
  const bool few = count <= n;
  const int per = (count + kWaves * 64 - 1) / (kWaves * 64) * 64;
  const int from = wave * per, to = min(count, from + per);
  int gt = 0, eq = 0;
  for (int i = from + lane; i - lane < to; i += 64) {
    const uint32_t k = i < to ? ranks[i] : 0;
    gt += __popcll(__ballot(few ? k > 0 : k > prefix));
    if (!few) eq += __popcll(__ballot(i < to && k == prefix && k > 0));
  }
  if (lane == 0) {
    s.gt[wave] = gt;
    s.eq[wave] = eq;
  }
  __syncthreads();
  int at = 0, ties = 0;
  for (int w = 0; w < wave; ++w) {
    at += s.gt[w] + min(s.eq[w], max(0, left - ties));
    ties += s.eq[w];
  }
  const uint64_t below = (uint64_t(1) << lane) - 1;
  for (int i = from + lane; i - lane < to; i += 64) {
    const uint32_t k = i < to ? ranks[i] : 0;
    const bool up = few ? k > 0 : k > prefix, tie = !few && i < to && k == prefix && k > 0;
    const uint64_t tied = __ballot(tie);
    const bool take = up || (tie && ties + __popcll(tied & below) < left);
    const uint64_t taken = __ballot(take);
    if (take) out[at + __popcll(taken & below)] = i;
    at += __popcll(taken);
    ties += __popcll(tied);
  }
  int all = 0, tied = 0;
  for (int w = 0; w < kWaves; ++w) {
    all += s.gt[w];
    tied += s.eq[w];
  }
  all += min(tied, left);
  for (int i = all + threadIdx.x; i < n; i += kThreads) out[i] = -1;
}

// Columns of a row that may be listed: up to its own block's.
__device__ __forceinline__ int columns(const KvSelectArgs& a, int64_t t, int* r, int* own) {
  *r = a.q.token_request[t];
  const int pos = a.q.positions[t];
  *own = pos >= 0 ? pos >> a.c.lps : -1;
  return *r >= 0 && *r < a.q.requests ? min(*own + 1, a.q.cols) : 0;
}

// A row's ranks in LDS, then its list.
template <bool BF16, int CH>
__global__ __launch_bounds__(kThreads) void kv_select_kernel(KvSelectArgs a) {
  extern __shared__ uint32_t ranks[];
  __shared__ Select s;
  __shared__ __align__(16) int8_t codes[kKvMaxDim];
  __shared__ float red[kWaves];
  const int h = (int)(blockIdx.x % a.c.heads);
  const int64_t t = blockIdx.x / a.c.heads;
  int r, own;
  const int count = columns(a, t, &r, &own);
  if (count > a.n) {  // (else every candidate is taken, whatever its score)
    query_codes<BF16>(a, t, h, codes, red);
    rank_columns<CH>(a, h, r, own, 0, count, codes, ranks);
  } else {
    for (int j = threadIdx.x; j < count; j += kThreads) {
      const int p = a.q.table[(int64_t)r * a.q.table_stride + j];
      ranks[j] = p >= 0 && p < a.c.pages ? kAlways : 0;
    }
  }
  __syncthreads();
  take_best(ranks, count, a.n, a.blocks + (t * a.c.heads + h) * a.n, s);
}

constexpr int kPartCols = 1024;

// Long rows: ranks to the workspace, a stretch of columns a workgroup ...
template <bool BF16, int CH>
__global__ __launch_bounds__(kThreads) void kv_select_ranks_kernel(KvSelectArgs a, int parts) {
  __shared__ __align__(16) int8_t codes[kKvMaxDim];
  __shared__ float red[kWaves];
  const int part = (int)(blockIdx.x % parts);
  const int64_t row = blockIdx.x / parts;
  const int h = (int)(row % a.c.heads);
  const int64_t t = row / a.c.heads;
  int r, own;
  const int count = columns(a, t, &r, &own);
  const int c0 = part * kPartCols, c1 = min(count, c0 + kPartCols);
  if (c0 >= c1) return;
  query_codes<BF16>(a, t, h, codes, red);
  rank_columns<CH>(a, h, r, own, c0, c1, codes, a.keys + row * a.q.cols + c0);
}

// ... and the lists from there.
__global__ __launch_bounds__(kThreads) void kv_select_lists_kernel(KvSelectArgs a) {
  __shared__ Select s;
  const int64_t row = blockIdx.x;
  int r, own;
  const int count = columns(a, row / a.c.heads, &r, &own);
  take_best(a.keys + row * a.q.cols, count, a.n, a.blocks + row * a.n, s);
}

bool in_lds(const KvSelectArgs& a) {
  return a.q.cols <= kLdsCols && (a.q.cols <= 4096 || a.q.tokens * a.c.heads >= 256);
}

template <bool BF16, int CH>
void launch_select(const KvSelectArgs& a, hipStream_t s) {
  const unsigned rows = (unsigned)(a.q.tokens * a.c.heads);
  if (in_lds(a)) {
    kv_select_kernel<BF16, CH><<<rows, kThreads, a.q.cols * 4, s>>>(a);
    return;
  }
  const int parts = (a.q.cols + kPartCols - 1) / kPartCols;
  kv_select_ranks_kernel<BF16, CH><<<rows * parts, kThreads, 0, s>>>(a, parts);
  kv_select_lists_kernel<<<rows, kThreads, 0, s>>>(a);
}

}  // namespace

int64_t kv_select_workspace(const KvSelectArgs& a) {
  return in_lds(a) ? 0 : a.q.tokens * a.c.heads * a.q.cols * 4;
}

int64_t kv_select_grid(const KvSelectArgs& a) {
  const int64_t rows = a.q.tokens * a.c.heads;
  return in_lds(a) ? rows : rows * ((a.q.cols + kPartCols - 1) / kPartCols);
}

hipError_t launch_kv_select(const KvSelectArgs& a, hipStream_t s) {
  if (a.c.dim % 16 == 0)
    a.c.bf16 ? launch_select<true, 16>(a, s) : launch_select<false, 16>(a, s);
  else
    a.c.bf16 ? launch_select<true, 8>(a, s) : launch_select<false, 8>(a, s);
  return hipGetLastError();
}

}  // namespace mlxvs::kern
