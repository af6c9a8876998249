// A step's block tables and slot maps from the requests' lengths.
//
// A request that holds `past` tokens and gets `fresh` more needs
// ceil((past + fresh) / page) - ceil(past / page) pages; a running sum over the
// requests says where in the free list they lie, another where its tokens lie
// in the step's batch.  A request is admitted if its columns suffice and the
// free list reaches to its last page (one that needs none, always): from the
// first request that the list cannot serve on, none takes pages.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "kv_cache.h"

namespace mlxvs::kern {
namespace {

struct Need {
  int64_t tokens, pages;
};

__device__ __forceinline__ Need operator+(Need x, Need y) {
  return {x.tokens + y.tokens, x.pages + y.pages};
}
__device__ __forceinline__ Need shfl_up(Need x, int by) {
  return {__shfl_up(x.tokens, by), __shfl_up(x.pages, by)};
}

struct Request {
  int64_t past, fresh, have, need;
  bool valid;
};

__device__ __forceinline__ Request request(const KvPlanArgs& a, int64_t r) {
  Request q{0, 0, 0, 0, false};
  if (r >= a.requests) return q;
  const int64_t past = a.past[r], fresh = a.fresh[r], page = int64_t(1) << a.lps;
  q.past = past;
  q.fresh = fresh > 0 ? fresh : 0;
  q.valid = past >= 0 && fresh >= 0 && past + fresh <= (int64_t(a.cols) << a.lps);
  if (q.valid) {
    q.have = (past + page - 1) >> a.lps;
    q.need = ((past + fresh + page - 1) >> a.lps) - q.have;
  }
  return q;
}

// Inclusive sums over a workgroup's THREADS threads; `all` gets the total.
template <int THREADS>
__device__ __forceinline__ Need scan(Need x, Need* waves, Need* all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int by = 1; by < 64; by <<= 1) {
    const Need y = shfl_up(x, by);
    if (lane >= by) x = x + y;
  }
  if (lane == 63) waves[wave] = x;
  __syncthreads();
  Need before{0, 0}, total{0, 0};
  for (int w = 0; w < THREADS / 64; ++w) {
    if (w < wave) before = before + waves[w];
    total = total + waves[w];
  }
  __syncthreads();
  *all = total;
  return x + before;
}

// A request's place among the others: its first token of the batch, and its
// first entry of the free list (-1: not admitted; one that takes no page: any).
struct Place {
  int32_t start, first;
};

__device__ __forceinline__ Place place(const Request& q, Need upto, int64_t cursor, int64_t left) {
  const bool admitted = q.valid && (q.need == 0 || upto.pages <= left);
  const int64_t start = upto.tokens - q.fresh;
  return {(int32_t)(start < INT32_MAX ? start : INT32_MAX),
          !admitted ? -1 : q.need ? (int32_t)(cursor + upto.pages - q.need) : 0};
}

__device__ __forceinline__ int64_t entries_left(const KvPlanArgs& a, int64_t cursor) {
  return cursor < 0 ? -1 : a.free_count - cursor;
}

// Token t of the batch, the requests' places being in `starts` and `first`.
__device__ __forceinline__ void token(const KvPlanArgs& a, int64_t t, const int32_t* starts,
                                      const int32_t* first) {
  const int64_t page = int64_t(1) << a.lps;
  int32_t who = -1, pos = -1;
  int64_t slot = -1;
  if (t < starts[a.requests]) {
    // the last request that starts at or before t (those without tokens start
    // where the next one does)
    int64_t lo = 0, hi = a.requests - 1;
    while (lo < hi) {
      const int64_t mid = (lo + hi + 1) / 2;
      if (starts[mid] <= t) lo = mid;
      else hi = mid - 1;
    }
    who = (int32_t)lo;
    const int32_t from = first[lo];
    if (from >= 0) {
      const int64_t past = a.past[lo];
      const int64_t at = past + t - starts[lo];
      const int64_t have = (past + page - 1) >> a.lps, col = at >> a.lps;
      const int32_t id = col < have ? a.table[lo * a.table_stride + col]
                                    : a.free_pages[from + col - have];
      pos = (int32_t)at;
      if (id >= 0) slot = ((int64_t)id << a.lps) + (at & (page - 1));
    }
  }
  a.slots[t] = slot;
  a.token_request[t] = who;
  a.positions[t] = pos;
}

// The new pages of request r, by one wavefront.
__device__ __forceinline__ void pages(const KvPlanArgs& a, int64_t r, int32_t first) {
  if (first < 0) return;
  const Request q = request(a, r);
  for (int64_t i = threadIdx.x & 63; i < q.need; i += 64)
    a.table[r * a.table_stride + q.have + i] = a.free_pages[first + i];
}

// Up to kFew requests: one launch, every workgroup taking the running sums of
// all requests for itself (8 bytes a request, from L2).  A thread sums a stretch
// of neighbouring requests.  In one and two launches 1,024 requests take 8.7 and
// 10.8 us with a token each, 11.9 and 11.8 with up to 63; 2,048 take 11.0 and
// 11.9, 20.7 and 16.4.  Few bytes: what bounds both is the chain of dependent
// accesses (lengths, cursor, free list, table).
constexpr int kFew = 1024;

__global__ __launch_bounds__(256) void kv_plan_kernel(KvPlanArgs a) {
  extern __shared__ int32_t places[];  // starts [requests + 1], first [requests]
  __shared__ Need waves[4];
  __shared__ unsigned long long taken;
  const int requests = (int)a.requests;
  int32_t *starts = places, *first = places + requests + 1;
  const int64_t cursor = a.cursor[0], left = entries_left(a, cursor);
  const bool writes = blockIdx.x == 0;
  if (threadIdx.x == 0) taken = 0;
  const int per = (requests + 255) / 256;
  const int r0 = min(requests, per * (int)threadIdx.x), r1 = min(requests, r0 + per);
  Need sum{0, 0}, all;
  for (int r = r0; r < r1; ++r) {
    const Request q = request(a, r);
    sum = sum + Need{q.fresh, q.need};
  }
  const Need upto = scan<256>(sum, waves, &all);
  Need at{upto.tokens - sum.tokens, upto.pages - sum.pages};
  for (int r = r0; r < r1; ++r) {
    const Request q = request(a, r);
    at = at + Need{q.fresh, q.need};
    const Place p = place(q, at, cursor, left);
    starts[r] = p.start;
    first[r] = p.first;
    if (writes) {
      a.starts[r] = p.start;
      a.first[r] = p.first;
      a.lengths[r] = (int32_t)(p.first < 0 ? q.past : q.past + q.fresh);
      if (p.first >= 0 && q.need) atomicMax(&taken, (unsigned long long)at.pages);
    }
  }
  if (threadIdx.x == 0)
    starts[requests] = (int32_t)(all.tokens < INT32_MAX ? all.tokens : INT32_MAX);
  __syncthreads();
  if (writes && threadIdx.x == 0) {
    a.starts[requests] = starts[requests];
    a.cursor_out[0] = (int32_t)(cursor + (int64_t)taken);
  }
  const int64_t grid = gridDim.x;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < a.tokens; t += grid * 256)
    token(a, t, starts, first);
  for (int64_t r = blockIdx.x + grid * (threadIdx.x >> 6); r < requests; r += 4 * grid)
    pages(a, r, first[r]);
}

// More: the running sums by one workgroup ...
constexpr int kThreads = 1024;

__global__ __launch_bounds__(kThreads) void kv_plan_requests_kernel(KvPlanArgs a) {
  __shared__ Need waves[kThreads / 64];
  __shared__ unsigned long long taken;
  if (threadIdx.x == 0) taken = 0;
  const int64_t cursor = a.cursor[0], left = entries_left(a, cursor);
  Need before{0, 0};
  for (int64_t r0 = 0; r0 < a.requests; r0 += kThreads) {
    const int64_t r = r0 + threadIdx.x;
    const Request q = request(a, r);
    Need all;
    const Need upto = before + scan<kThreads>({q.fresh, q.need}, waves, &all);
    if (r < a.requests) {
      const Place p = place(q, upto, cursor, left);
      a.starts[r] = p.start;
      a.first[r] = p.first;
      a.lengths[r] = (int32_t)(p.first < 0 ? q.past : q.past + q.fresh);
      if (p.first >= 0 && q.need) atomicMax(&taken, (unsigned long long)upto.pages);
    }
    before = before + all;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    a.starts[a.requests] = (int32_t)(before.tokens < INT32_MAX ? before.tokens : INT32_MAX);
    a.cursor_out[0] = (int32_t)(cursor + (int64_t)taken);
  }
}

// ... then tokens and new pages: the first workgroups a token a thread, the
// others a request a wavefront.
__global__ __launch_bounds__(256) void kv_plan_tokens_kernel(KvPlanArgs a, int64_t token_blocks) {
  if (blockIdx.x < token_blocks) {
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (t < a.tokens) token(a, t, a.starts, a.first);
    return;
  }
  const int64_t r = ((int64_t)blockIdx.x - token_blocks) * 4 + (threadIdx.x >> 6);
  if (r < a.requests) pages(a, r, a.first[r]);
}

}  // namespace

hipError_t launch_kv_plan(const KvPlanArgs& a, hipStream_t s) {
  const int64_t token_blocks = (a.tokens + 255) / 256;
  if (a.requests <= kFew) {
    const int64_t grid =
        std::max<int64_t>(1, std::min<int64_t>(512, std::max(token_blocks, (a.requests + 15) / 16)));
    kv_plan_kernel<<<dim3((unsigned)grid), 256, (2 * a.requests + 1) * 4, s>>>(a);
    return hipGetLastError();
  }
  kv_plan_requests_kernel<<<1, kThreads, 0, s>>>(a);
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  const int64_t blocks = token_blocks + (a.requests + 3) / 4;
  kv_plan_tokens_kernel<<<dim3((unsigned)blocks), 256, 0, s>>>(a, token_blocks);
  return hipGetLastError();
}

}  // namespace mlxvs::kern
