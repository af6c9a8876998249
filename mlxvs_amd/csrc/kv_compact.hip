// Requests cut to the tokens that a budget leaves: slot j of a request and kv head
// gets key, value and mass of slot kept[j], in place and in order, the complete
// pages that hold other tokens now get their summaries anew, and the pages past the
// new end go back into the free list.
//
// The lists ascend, so kept[j] >= j.  A workgroup moves a tile of slots: it reads
// all that comes there into registers, says so, waits until the tiles before it that
// have slots of its own as their sources have said so too, and writes.  Reads wait
// for nothing, and workgroups take their tiles in order, by a counter: whoever is
// waited for has been running since before the one that waits.  It moves bytes, each
// read once and written once; a second copy, from which tiles could be taken in any
// order, would double that.  Measured: 32 requests of up to 16,384 tokens, 8 heads of
// 128 values, cut to 4,096, 281 us (tile after tile by one workgroup a row 1,610); two
// of 60,001 cut to 40,009 in pages of 16, 3 heads of 80, 51 (8,047).  Values lie
// transposed in their pages, so where a part of a page's tokens is kept all its lines
// are read: 1.35 GB instead of 0.88 in the first case, 4.8 TB/s.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "kv_cache.h"
#include "kv_summary.h"
#include "kv_values.h"

namespace mlxvs::kern {
namespace {

constexpr int kTile = 128;  // slots of a workgroup
constexpr int kThreads = 256;
constexpr int kPlanThreads = 1024;
constexpr int kPagesOfTile = kTile / 16;

// The workspace: the counter of tiles taken, the number of requests that are cut,
// these, where each one's pages go in the free list, and a flag for each tile of a
// request and head: what comes there has been read.
struct Work {
  uint32_t* taken;
  int32_t* count;
  int32_t* who;    // [requests]
  int32_t* place;  // [requests]
  uint32_t* read;  // [cut requests][heads][tiles]
};
constexpr int kFlags = 64;  // (the counter has a line of its own)

__host__ __device__ __forceinline__ int tiles_of(const KvCompactArgs& a) {
  return (int)(((int64_t)a.n + kTile - 1) / kTile);
}
__device__ __forceinline__ Work work_of(const KvCompactArgs& a) {
  int32_t* w = a.work;
  return {(uint32_t*)w, w + 32, w + kFlags, w + kFlags + a.requests,
          (uint32_t*)(w + kFlags + 2 * a.requests)};
}

// Which requests are cut, and the free list: a running sum over the requests of the
// pages that each gives back, from the cursor down.  The list has room for what
// was taken from it; from the first request whose pages it has not on, none that
// gives pages back is cut.  By the first workgroup; the others clear the flags.
__global__ __launch_bounds__(kPlanThreads) void kv_compact_plan_kernel(KvCompactArgs a) {
  __shared__ int64_t waves[kPlanThreads / 64];
  __shared__ int cuts[kPlanThreads / 64];
  __shared__ unsigned long long given;
  const Work work = work_of(a);
  if (blockIdx.x > 0) {
    const int64_t flags = a.requests * a.c.heads * tiles_of(a);
    const int64_t step = (int64_t)(gridDim.x - 1) * kPlanThreads;
    for (int64_t i = (int64_t)(blockIdx.x - 1) * kPlanThreads + threadIdx.x; i < flags; i += step)
      work.read[i] = 0;
    return;
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (threadIdx.x == 0) {
    given = 0;
    work.taken[0] = 0;
  }
  const int64_t cursor = a.cursor[0], page = int64_t(1) << a.c.lps;
  const int64_t room = cursor <= a.free_count ? cursor : -1;
  const int64_t want = (a.n + page - 1) >> a.c.lps;
  int64_t before = 0;
  int count = 0;
  for (int64_t r0 = 0; r0 < a.requests; r0 += kPlanThreads) {
    const int64_t r = r0 + threadIdx.x;
    int64_t length = 0, frees = 0;
    bool cut = false;
    if (r < a.requests) {
      length = a.lengths[r];
      cut = length > a.n && length <= (int64_t(a.cols) << a.c.lps) &&
            a.kept[r * a.c.heads * a.n] >= 0;
      if (cut) frees = ((length + page - 1) >> a.c.lps) - want;
    }
    int64_t upto = frees;
#pragma unroll
    for (int by = 1; by < 64; by <<= 1) {
      const int64_t y = __shfl_up(upto, by);
      if (lane >= by) upto += y;
    }
    if (lane == 63) waves[wave] = upto;
    __syncthreads();
    int64_t all = 0;
    for (int w = 0; w < kPlanThreads / 64; ++w) {
      if (w < wave) upto += waves[w];
      all += waves[w];
    }
    upto += before;
    before += all;
    cut = cut && (frees == 0 || upto <= room);
    const uint64_t some = __ballot(cut);
    if (lane == 0) cuts[wave] = (int)__popcll(some);
    __syncthreads();
    int at = count + (int)__popcll(some & ((uint64_t(1) << lane) - 1));
    for (int w = 0; w < kPlanThreads / 64; ++w) {
      if (w < wave) at += cuts[w];
      count += cuts[w];
    }
    if (r < a.requests) a.lengths_out[r] = (int32_t)(cut ? a.n : length);
    if (cut) {
      work.who[at] = (int32_t)r;
      work.place[at] = (int32_t)(cursor - upto);
      if (frees) atomicMax(&given, (unsigned long long)upto);
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    a.cursor_out[0] = (int32_t)(cursor - (int64_t)given);
    work.count[0] = count;
  }
}

// Waits until the tiles before `tile` that have some of its slots as their sources
// have been read: those whose last source reaches it, the ones right before it.  By
// one wavefront.  (Nothing of what they read is needed here, and their loads were
// complete before they said so: the flag alone is waited for.)
__device__ __forceinline__ void wait_for_readers(const int32_t* kept, const uint32_t* read,
                                                 int tile, int lane) {
  for (int from = tile - 1; from >= 0; from -= 64) {
    const int t = from - lane;
    const bool needed = t >= 0 && kept[t * kTile + kTile - 1] >= tile * kTile;
    bool missing = needed;
    while (__any(missing)) {
      if (missing)
        missing = __hip_atomic_load(read + t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == 0;
    }
    if (!__all(needed)) return;
  }
}

// The summaries of a tile's pages (of at most kTile tokens) from its keys in registers.
// Two neighbouring values' sums are one number, x + 2^16 y (128 codes of up to 127 stay
// below 2^15): half as many additions in LDS (the two of 60,001 53 -> 51 us).
struct TileSums {
  uint32_t top[kPagesOfTile];  // the largest |value|, as bits
  int bad[kPagesOfTile];       // some value is not finite
  int sum[kPagesOfTile][kKvMaxDim / 2];
};
static_assert(kTile * 127 < 1 << 15);

template <bool BF16, int N>
__device__ __forceinline__ void tile_summaries(const KvCompactArgs& a, TileSums& s,
                                               const uintx4 (&k)[N], const int64_t* to_page,
                                               const int* wanted, int pages) {
  const int tid = threadIdx.x, d = a.c.dim, chunks = d / 8, lps = a.c.lps;
  for (int i = tid; i < pages; i += kThreads) s.top[i] = s.bad[i] = 0;
  for (int i = tid; i < pages * (kKvMaxDim / 2); i += kThreads) (&s.sum[0][0])[i] = 0;
  __syncthreads();
#pragma unroll
  for (int x = 0; x < N; ++x) {
    const int i = tid + kThreads * x, p = i / chunks >> lps;
    const bool mine = p < pages && wanted[p];
    float top = 0.0f;
    bool bad = false;
    if (mine) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float v = fabsf(value<BF16>(k[x], j));
        bad |= !(v < __builtin_inff());
        top = fmaxf(top, v);
      }
    }
    // (neighbouring lanes mostly have one page)
    const int first = __builtin_amdgcn_readfirstlane(p);
    if (__all(p == first)) {
      top = wave_max(top);
      bad = __any(bad);
      if (mine && (tid & 63) == 0) {
        atomicMax(&s.top[p], __builtin_bit_cast(uint32_t, top));
        if (bad) s.bad[p] = 1;
      }
    } else if (mine) {
      atomicMax(&s.top[p], __builtin_bit_cast(uint32_t, top));
      if (bad) s.bad[p] = 1;
    }
  }
  __syncthreads();
#pragma unroll
  for (int x = 0; x < N; ++x) {
    const int i = tid + kThreads * x, p = i / chunks >> lps;
    if (p >= pages || !wanted[p] || s.bad[p]) continue;
    const float top = __builtin_bit_cast(float, s.top[p]);
    if (!(top > 1e-30f)) continue;
    const float inv = 127.0f / top;
#pragma unroll
    for (int j = 0; j < 8; j += 2)
      atomicAdd(&s.sum[p][4 * (i % chunks) + j / 2], (int)rintf(value<BF16>(k[x], j) * inv) +
                                                         (int)rintf(value<BF16>(k[x], j + 1) * inv) * 65536);
  }
  __syncthreads();
  const int lane = tid & 63;
  for (int p = tid >> 6; p < pages; p += kThreads / 64) {
    if (!wanted[p]) continue;
    const int64_t at = to_page[p << lps];
    if (at < 0) continue;
    const auto sum = [&](int i) {
      const int both = s.sum[p][i / 2], first = (int16_t)both;
      return (float)(i % 2 ? (both - first) / 65536 : first);
    };
    float peak = 0.0f;
    for (int i = lane; i < d; i += 64) peak = fmaxf(peak, fabsf(sum(i)));
    peak = wave_max(peak);
    const float to = peak > 0.0f ? 127.0f / peak : 0.0f;
    for (int i = lane; i < d; i += 64) a.c.summaries[at * d + i] = (int8_t)rintf(sum(i) * to);
    const float top = __builtin_bit_cast(float, s.top[p]);
    if (lane == 0)
      a.c.scales[at] = s.bad[p]          ? __builtin_inff()
                       : !(top > 1e-30f) ? 0.0f
                                         : top * (peak / (16129.0f * (float)a.c.page));
  }
}

// DP: head size rounded up.
template <int DP, bool BF16>
__global__ __launch_bounds__(kThreads, 2) void kv_compact_kernel(KvCompactArgs a) {
  constexpr int kK = kTile * DP / 8 / kThreads;  // 16-byte pieces of keys a thread
  constexpr int kV = kTile / 2 * DP / kThreads;  // pairs of slots' values a thread
  __shared__ int64_t from_page[kTile], to_page[kTile];
  __shared__ int from_off[kTile], to_off[kTile];
  __shared__ int wanted[kPagesOfTile];
  __shared__ int ticket, other, moves;  // (some slot changes, some key and value)
  __shared__ TileSums sums;
  const Work work = work_of(a);
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t rows = (int64_t)work.count[0] * a.c.heads;
  if (blockIdx.x >= rows * tiles_of(a)) return;
  if (tid == 0) {
    ticket = (int)__hip_atomic_fetch_add(work.taken, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    other = moves = 0;
  }
  if (tid < kPagesOfTile) wanted[tid] = 0;
  __syncthreads();
  // the first tiles of all rows, then the second ones
  const int tile = (int)(ticket / rows);
  const int64_t row = ticket % rows;
  const int h = (int)(row % a.c.heads), cut = (int)(row / a.c.heads);
  const int64_t r = work.who[cut];
  const int32_t* table = a.table + r * a.table_stride;
  const int32_t* kept = a.kept + (r * a.c.heads + h) * a.n;
  float* mass = a.mass ? a.mass + (r * a.c.heads + h) * a.slots : nullptr;
  uint32_t* read = work.read + row * tiles_of(a);
  const int d = a.c.dim, lps = a.c.lps, page = a.c.page, chunks = d / 8;
  const int j0 = tile * kTile, count = min(kTile, a.n - j0);
  const int64_t head = (int64_t)page * d;

  if (tile == 0 && h == 0) {
    const int want = (a.n + page - 1) >> lps, have = (a.lengths[r] + page - 1) >> lps;
    for (int i = tid; i < have - want; i += kThreads)
      a.free_pages[work.place[cut] + i] = table[want + i];
  }
  float m = 0.0f;
  if (tid < kTile) {
    const int src = tid < count ? kept[j0 + tid] : -1, dst = j0 + tid;
    const auto place = [&](int slot) {  // page x heads + head, -1: absent
      const int p = slot >= 0 && slot >> lps < a.cols ? table[slot >> lps] : -1;
      return p >= 0 && p < a.c.pages ? (int64_t)p * a.c.heads + h : -1;
    };
    const int64_t from = place(src), to = src >= 0 ? place(dst) : -1;
    // (a key that does not come leaves what is there)
    from_page[tid] = from >= 0 ? from : to;
    from_off[tid] = (from >= 0 ? src : dst) & (page - 1);
    to_page[tid] = to;
    to_off[tid] = from >= 0 && to >= 0 && src != dst ? dst & (page - 1) : -1;
    if (to_off[tid] >= 0) moves = 1;
    if (src >= 0 && src != dst) {
      other = 1;
      if (page <= kTile && (j0 >> lps) + (tid >> lps) < a.n >> lps) wanted[tid >> lps] = 1;
    }
    if (mass && src >= 0) m = mass[min((int64_t)src, a.slots - 1)];
  }
  __syncthreads();
  uintx4 k[kK];
  uint16_t v[kV][2];
  // two neighbouring slots' values a thread
  const int jv = 2 * (tid % (kTile / 2)), iv = tid / (kTile / 2);
  constexpr int kStepV = kThreads / (kTile / 2);
  if (moves) {
    // (all loads are in flight together: none has a condition, and what is not
    // written is read from a place that is there)
#pragma unroll
    for (int x = 0; x < kK; ++x) {
      const int i = tid + kThreads * x, j = min(i / chunks, kTile - 1);
      k[x] = *(const uintx4*)((const uint16_t*)a.c.keys + max((int64_t)0, from_page[j]) * head +
                              from_off[j] * d + 8 * (i % chunks));
    }
    const uint16_t *src[2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
      src[u] = (const uint16_t*)a.c.values + max((int64_t)0, from_page[jv + u]) * head + from_off[jv + u];
#pragma unroll
    for (int x = 0; x < kV; ++x) {
      const int i = min(iv + kStepV * x, d - 1) * page;
#pragma unroll
      for (int u = 0; u < 2; ++u) v[x][u] = src[u][i];
    }
  }
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // all of it is here
#endif
  __syncthreads();
  if (tid == 0) __hip_atomic_store(read + tile, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  if (!other) return;
  if (tid < 64) wait_for_readers(kept, read, tile, lane);
  __syncthreads();
  if (moves) {
#pragma unroll
    for (int x = 0; x < kK; ++x) {
      const int i = tid + kThreads * x, j = i / chunks;
      if (j < kTile && to_off[j] >= 0)
        *(uintx4*)((uint16_t*)a.c.keys + to_page[j] * head + to_off[j] * d + 8 * (i % chunks)) = k[x];
    }
    // (two neighbouring slots are in one page)
    const bool u0 = to_off[jv] >= 0, u1 = to_off[jv + 1] >= 0;
    uint16_t* to = (uint16_t*)a.c.values + to_page[u0 ? jv : jv + 1] * head + ((j0 + jv) & (page - 1));
#pragma unroll
    for (int x = 0; x < kV; ++x) {
      const int i = iv + kStepV * x;
      if (i >= d) continue;
      if (u0 && u1) *(uint32_t*)(to + i * page) = v[x][0] | (uint32_t)v[x][1] << 16;
      else if (u0) to[i * page] = v[x][0];
      else if (u1) to[i * page + 1] = v[x][1];
    }
  }
  if (mass && tid < count) mass[j0 + tid] = m;
  if (a.c.summaries && page <= kTile && moves) {
    const int pages = (a.n >> lps) - (j0 >> lps);  // complete ones from here on
    if (pages > 0)
      tile_summaries<BF16>(a, sums, k, to_page, wanted, min(pages, kTile >> lps));
  }
}

// Pages of more tokens than a tile: a complete page and head of a request that was
// cut.
template <bool BF16>
__global__ __launch_bounds__(64) void kv_compact_summaries_kernel(KvCompactArgs a, int pages) {
  __shared__ Sums sums;
  const Work work = work_of(a);
  const int h = (int)(blockIdx.x % a.c.heads);
  const int64_t rest = blockIdx.x / a.c.heads;
  const int col = (int)(rest % pages);
  if (rest / pages >= work.count[0]) return;
  const int64_t r = work.who[rest / pages];
  const int32_t* kept = a.kept + (r * a.c.heads + h) * a.n + ((int64_t)col << a.c.lps);
  bool other = false;
  for (int i = threadIdx.x; i < a.c.page; i += 64) other |= kept[i] != (col << a.c.lps) + i;
  if (!__any(other)) return;
  const int p = a.table[r * a.table_stride + col];
  if (p < 0 || p >= a.c.pages) return;
  const int64_t at = (int64_t)p * a.c.heads + h;
  const uint16_t* held = (const uint16_t*)a.c.keys + at * a.c.page * a.c.dim;
  summarise<BF16, 64>(a.c, at, sums, [&](int i) { return held + i * a.c.dim; });
}

template <int DP>
void launch_move(const KvCompactArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)(a.requests * a.c.heads * tiles_of(a)));
  if (a.c.bf16) kv_compact_kernel<DP, true><<<grid, kThreads, 0, s>>>(a);
  else kv_compact_kernel<DP, false><<<grid, kThreads, 0, s>>>(a);
}

}  // namespace

int64_t kv_compact_workspace(const KvCompactArgs& a) {
  const int64_t ints = kFlags + 2 * a.requests + a.requests * a.c.heads * tiles_of(a);
  return (ints * 4 + 15) / 16 * 16;
}

int64_t kv_compact_grid(const KvCompactArgs& a) { return a.requests * a.c.heads * tiles_of(a); }

hipError_t launch_kv_compact(const KvCompactArgs& a, hipStream_t s) {
  const int64_t flags = a.requests * a.c.heads * tiles_of(a);
  const unsigned clear = (unsigned)std::min<int64_t>(256, (flags + kPlanThreads - 1) / kPlanThreads);
  kv_compact_plan_kernel<<<1 + clear, kPlanThreads, 0, s>>>(a);
  if (hipError_t e = hipGetLastError(); e != hipSuccess || a.requests == 0) return e;
  if (a.c.dim <= 64) launch_move<64>(a, s);
  else if (a.c.dim <= 96) launch_move<96>(a, s);
  else if (a.c.dim <= 128) launch_move<128>(a, s);
  else if (a.c.dim <= 192) launch_move<192>(a, s);
  else launch_move<256>(a, s);
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  const int pages = a.n >> a.c.lps;
  if (!a.c.summaries || pages == 0 || a.c.page <= kTile) return hipSuccess;
  const dim3 grid((unsigned)(a.requests * a.c.heads * pages));
  if (a.c.bf16) kv_compact_summaries_kernel<true><<<grid, 64, 0, s>>>(a, pages);
  else kv_compact_summaries_kernel<false><<<grid, 64, 0, s>>>(a, pages);
  return hipGetLastError();
}

}  // namespace mlxvs::kern
