// Requests cut to the tokens that a budget leaves: slot j of a request and kv head
// gets key, value and mass of slot kept[j], in place and in order, the complete
// pages that hold other tokens now get their summaries anew, and the pages past the
// new end go back into the free list.
//
// The lists ascend, so kept[j] >= j: tiles of slots are moved from the first to the
// last, each read whole before it is written, and none is written before those that
// come from it have been read.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "kv_cache.h"
#include "kv_summary.h"
#include "kv_values.h"

namespace mlxvs::kern {
namespace {

constexpr int kTile = 64;  // slots
constexpr int kPlanThreads = 1024;

// Which requests are cut, and the free list: a running sum over the requests of the
// pages that each gives back, from the cursor down.  The list has room for what
// was taken from it; from the first request whose pages it has not on, none that
// gives pages back is cut.
__global__ __launch_bounds__(kPlanThreads) void kv_compact_plan_kernel(KvCompactArgs a) {
  __shared__ int64_t waves[kPlanThreads / 64];
  __shared__ unsigned long long given;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (threadIdx.x == 0) given = 0;
  const int64_t cursor = a.cursor[0], page = int64_t(1) << a.c.lps;
  const int64_t room = cursor <= a.free_count ? cursor : -1;
  const int64_t want = (a.n + page - 1) >> a.c.lps;
  int64_t before = 0;
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
    if (r < a.requests) {
      a.cut[r] = cut;
      a.lengths_out[r] = (int32_t)(cut ? a.n : length);
      if (cut && frees) atomicMax(&given, (unsigned long long)upto);
    }
    // a wavefront gives back the pages of its 64 requests
    for (uint64_t todo = __ballot(cut && frees > 0); todo; todo &= todo - 1) {
      const int x = __builtin_ctzll(todo);
      const int64_t who = __shfl(r, x), count = __shfl(frees, x), at = cursor - __shfl(upto, x);
      for (int64_t i = lane; i < count; i += 64)
        a.free_pages[at + i] = a.table[who * a.table_stride + want + i];
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) a.cursor_out[0] = (int32_t)(cursor - (int64_t)given);
}

// A slot of a request and head: its page's and its own place there, absent pages -1.
struct Place {
  int64_t page;  // page x heads + head
  int off;
};
__device__ __forceinline__ Place place_of(const KvCompactArgs& a, const int32_t* table, int h,
                                          int slot) {
  const int col = slot >> a.c.lps;
  const int p = slot >= 0 && col < a.cols ? table[col] : -1;
  return {p >= 0 && p < a.c.pages ? (int64_t)p * a.c.heads + h : -1, slot & (a.c.page - 1)};
}

// A request and head.
__global__ __launch_bounds__(256) void kv_compact_kernel(KvCompactArgs a) {
  __shared__ int64_t from_page[kTile], to_page[kTile];
  __shared__ int from_off[kTile], to_off[kTile];
  const int h = (int)(blockIdx.x % a.c.heads);
  const int64_t r = blockIdx.x / a.c.heads;
  if (!a.cut[r]) return;
  const int32_t* table = a.table + r * a.table_stride;
  const int32_t* kept = a.kept + (int64_t)blockIdx.x * a.n;
  float* mass = a.mass ? a.mass + (int64_t)blockIdx.x * a.slots : nullptr;
  const int d = a.c.dim, page = a.c.page, chunks = d / 8, tid = threadIdx.x;
  const int64_t head = (int64_t)page * d;
  constexpr int kMostK = kTile * kKvMaxDim / 8 / 256, kMostV = kTile * kKvMaxDim / 256;
  for (int j0 = 0; j0 < a.n; j0 += kTile) {
    const int count = min(kTile, a.n - j0);
    if (tid < kTile) {
      const int src = tid < count ? kept[j0 + tid] : -1;
      const Place f = place_of(a, table, h, src), t = place_of(a, table, h, j0 + tid);
      from_page[tid] = f.page;
      from_off[tid] = f.off;
      to_page[tid] = tid < count && f.page >= 0 ? t.page : -1;
      to_off[tid] = t.off;
    }
    __syncthreads();
    uintx4 k[kMostK];
    uint16_t v[kMostV];
    float m = 0.0f;
#pragma unroll
    for (int x = 0; x < kMostK; ++x) {
      const int i = tid + 256 * x, j = i / chunks;
      if (j < kTile && to_page[j] >= 0)
        k[x] = *(const uintx4*)((const uint16_t*)a.c.keys + from_page[j] * head + from_off[j] * d +
                                8 * (i % chunks));
    }
    const int j = tid % kTile;
#pragma unroll
    for (int x = 0; x < kMostV; ++x) {
      const int i = tid / kTile + 256 / kTile * x;
      if (i < d && to_page[j] >= 0)
        v[x] = ((const uint16_t*)a.c.values)[from_page[j] * head + i * page + from_off[j]];
    }
    if (mass && tid < count) m = mass[min((int64_t)max(0, kept[j0 + tid]), a.slots - 1)];
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    __syncthreads();
#pragma unroll
    for (int x = 0; x < kMostK; ++x) {
      const int i = tid + 256 * x, jk = i / chunks;
      if (jk < kTile && to_page[jk] >= 0)
        *(uintx4*)((uint16_t*)a.c.keys + to_page[jk] * head + to_off[jk] * d + 8 * (i % chunks)) =
            k[x];
    }
#pragma unroll
    for (int x = 0; x < kMostV; ++x) {
      const int i = tid / kTile + 256 / kTile * x;
      if (i < d && to_page[j] >= 0)
        ((uint16_t*)a.c.values)[to_page[j] * head + i * page + to_off[j]] = v[x];
    }
    if (mass && tid < count) mass[j0 + tid] = m;
    __syncthreads();
  }
}

// A complete page and head of a request that was cut.
template <bool BF16>
__global__ __launch_bounds__(64) void kv_compact_summaries_kernel(KvCompactArgs a, int pages) {
  __shared__ Sums sums;
  const int h = (int)(blockIdx.x % a.c.heads);
  const int64_t rest = blockIdx.x / a.c.heads;
  const int col = (int)(rest % pages);
  const int64_t r = rest / pages;
  if (!a.cut[r]) return;
  const int32_t* kept = a.kept + (r * a.c.heads + h) * a.n + ((int64_t)col << a.c.lps);
  bool other = false;
  for (int i = threadIdx.x; i < a.c.page; i += 64) other |= kept[i] != (col << a.c.lps) + i;
  if (!__any(other)) return;
  const Place p = place_of(a, a.table + r * a.table_stride, h, col << a.c.lps);
  if (p.page < 0) return;
  const uint16_t* held = (const uint16_t*)a.c.keys + p.page * a.c.page * a.c.dim;
  summarise<BF16, 64>(a.c, p.page, sums, [&](int i) { return held + i * a.c.dim; });
}

}  // namespace

int64_t kv_compact_workspace(const KvCompactArgs& a) { return (a.requests * 4 + 15) / 16 * 16; }

int64_t kv_compact_grid(const KvCompactArgs& a) {
  return a.requests * a.c.heads * std::max<int64_t>(1, a.c.summaries ? a.n >> a.c.lps : 0);
}

hipError_t launch_kv_compact(const KvCompactArgs& a, hipStream_t s) {
  kv_compact_plan_kernel<<<1, kPlanThreads, 0, s>>>(a);
  if (hipError_t e = hipGetLastError(); e != hipSuccess || a.requests == 0) return e;
  kv_compact_kernel<<<dim3((unsigned)(a.requests * a.c.heads)), 256, 0, s>>>(a);
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  const int pages = a.n >> a.c.lps;
  if (!a.c.summaries || pages == 0) return hipSuccess;
  const dim3 grid((unsigned)(a.requests * a.c.heads * pages));
  if (a.c.bf16) kv_compact_summaries_kernel<true><<<grid, 64, 0, s>>>(a, pages);
  else kv_compact_summaries_kernel<false><<<grid, 64, 0, s>>>(a, pages);
  return hipGetLastError();
}

}  // namespace mlxvs::kern
