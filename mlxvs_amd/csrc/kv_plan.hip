// A step's block tables and slot maps from the requests' lengths.
//
// A request that holds `past` tokens and gets `fresh` more needs
// ceil((past + fresh) / page) - ceil(past / page) pages; a running sum over the
// requests says where in the free list they lie, another where its tokens lie
// in the step's batch.  A request is admitted if its columns suffice and the
// free list reaches to its last page (one that needs none, always): from the
// first request that the list cannot serve on, none takes pages.
#include <hip/hip_runtime.h>

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

constexpr int kThreads = 1024;

// Inclusive sums over a workgroup's threads; `all` gets the workgroup's total.
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
  for (int w = 0; w < kThreads / 64; ++w) {
    if (w < wave) before = before + waves[w];
    total = total + waves[w];
  }
  __syncthreads();
  *all = total;
  return x + before;
}

// The running sums, by one workgroup.
__global__ __launch_bounds__(kThreads) void kv_plan_requests_kernel(KvPlanArgs a) {
  __shared__ Need waves[kThreads / 64];
  __shared__ unsigned long long taken;
  if (threadIdx.x == 0) taken = 0;
  const int64_t cursor = a.cursor[0];
  const int64_t left = cursor < 0 ? -1 : a.free_count - cursor;
  Need before{0, 0};
  for (int64_t r0 = 0; r0 < a.requests; r0 += kThreads) {
    const int64_t r = r0 + threadIdx.x;
    const Request q = request(a, r);
    Need all;
    const Need upto = before + scan({q.fresh, q.need}, waves, &all);
    if (r < a.requests) {
      const bool admitted = q.valid && (q.need == 0 || upto.pages <= left);
      const int64_t start = upto.tokens - q.fresh;
      a.starts[r] = (int32_t)(start < INT32_MAX ? start : INT32_MAX);
      a.lengths[r] = (int32_t)(admitted ? q.past + q.fresh : q.past);
      // (a request that takes none: any entry says that it is admitted)
      a.first[r] = !admitted ? -1 : q.need ? (int32_t)(cursor + upto.pages - q.need) : 0;
      if (admitted && q.need) atomicMax(&taken, (unsigned long long)upto.pages);
    }
    before = before + all;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    a.starts[a.requests] = (int32_t)(before.tokens < INT32_MAX ? before.tokens : INT32_MAX);
    a.cursor_out[0] = (int32_t)(cursor + (int64_t)taken);
  }
}

// Tokens and new pages: the first workgroups a token a thread, the others a
// request a wavefront.
__global__ __launch_bounds__(256) void kv_plan_tokens_kernel(KvPlanArgs a, int64_t token_blocks) {
  const int64_t page = int64_t(1) << a.lps;
  if (blockIdx.x < token_blocks) {
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (t >= a.tokens) return;
    int32_t who = -1, pos = -1;
    int64_t slot = -1;
    if (t < a.starts[a.requests]) {
      // the last request that starts at or before t (those without tokens
      // start where the next one does)
      int64_t lo = 0, hi = a.requests - 1;
      while (lo < hi) {
        const int64_t mid = (lo + hi + 1) / 2;
        if (a.starts[mid] <= t) lo = mid;
        else hi = mid - 1;
      }
      who = (int32_t)lo;
      const int32_t first = a.first[lo];
      if (first >= 0) {
        const int64_t past = a.past[lo];
        const int64_t at = past + t - a.starts[lo];
        const int64_t have = (past + page - 1) >> a.lps, col = at >> a.lps;
        const int32_t id = col < have ? a.table[lo * a.table_stride + col]
                                      : a.free_pages[first + col - have];
        pos = (int32_t)at;
        if (id >= 0) slot = ((int64_t)id << a.lps) + (at & (page - 1));
      }
    }
    a.slots[t] = slot;
    a.token_request[t] = who;
    a.positions[t] = pos;
    return;
  }
  const int64_t r = ((int64_t)blockIdx.x - token_blocks) * 4 + (threadIdx.x >> 6);
  if (r >= a.requests) return;
  const int32_t first = a.first[r];
  if (first < 0) return;
  const Request q = request(a, r);
  for (int64_t i = threadIdx.x & 63; i < q.need; i += 64)
    a.table[r * a.table_stride + q.have + i] = a.free_pages[first + i];
}

}  // namespace

hipError_t launch_kv_plan(const KvPlanArgs& a, hipStream_t s) {
  kv_plan_requests_kernel<<<1, kThreads, 0, s>>>(a);
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  const int64_t token_blocks = (a.tokens + 255) / 256;
  const int64_t blocks = token_blocks + (a.requests + 3) / 4;
  if (blocks > 0)
    kv_plan_tokens_kernel<<<dim3((unsigned)blocks), 256, 0, s>>>(a, token_blocks);
  return hipGetLastError();
}

}  // namespace mlxvs::kern
