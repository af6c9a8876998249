// Host side of the paged key-value cache: argument checks, the kernels'
// argument blocks, and the C++ API of include/mlxvs/mlxvs.hpp.  The calls
// allocate nothing and keep no state, so unlike the search entries they need no
// per-device lock and no order among themselves.
#include <hip/hip_runtime.h>

#include <cmath>
#include <stdexcept>
#include <string>

#include "kv_cache.h"
#include "mlxvs/mlxvs.hpp"
#include "stage.h"

namespace mlxvs {
namespace {

// A check of a call's arguments; errors name the call.
struct Check {
  const char* op;
  void operator()(bool ok, const char* what) const {
    if (!ok) throw std::invalid_argument(std::string("[") + op + "] " + what);
  }
};

constexpr int64_t kIntMax = (int64_t(1) << 31) - 1;

bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

int log2_page(int32_t page_size, const Check& check) {
  for (int l = 4; l <= 8; ++l)
    if (page_size == 1 << l) return l;
  check(false, "page_size must be 16, 32, 64, 128 or 256.");
  return 0;
}

// A launch of `blocks` workgroups of `threads`.
void check_grid(int64_t blocks, int threads, const Check& check) {
  check(blocks * threads < (int64_t(1) << 32), "too many tokens for one call.");
}

kern::KvCache cache_of(const KvCache& c, const Check& check) {
  const int lps = log2_page(c.page_size, check);
  check(c.dim >= 8 && c.dim <= kern::kKvMaxDim && c.dim % 8 == 0,
        "dim must be a multiple of 8 in [8, 256].");
  check(c.heads >= 1 && c.heads <= 1 << 16, "heads must be in [1, 65536].");
  check(c.pages >= 0 && c.pages <= kIntMax, "pages must be in [0, 2^31).");
  check((c.summaries == nullptr) == (c.scales == nullptr),
        "summaries and scales come together.");
  check(c.pages == 0 || (c.keys != nullptr && c.values != nullptr),
        "keys and values must not be NULL.");
  check(aligned(c.keys) && aligned(c.values) && aligned(c.summaries),
        "keys, values and summaries must be 16-byte aligned.");
  return {c.keys,  c.values, c.summaries, c.scales, c.pages,
          c.heads, c.dim,    c.page_size, lps,      c.type == KvType::BFloat16};
}

kern::KvQueries queries_of(const KvQueries& q, const kern::KvCache& c, const Check& check) {
  check(q.tokens >= 0 && q.requests >= 0 && q.requests <= kIntMax && q.columns >= 0,
        "tokens, requests and columns must not be negative.");
  check(q.q_heads >= c.heads && q.q_heads % c.heads == 0 && q.q_heads <= 1 << 20,
        "q_heads must be a multiple of the cache's heads.");
  check(((int64_t)q.columns << c.lps) <= kIntMax, "columns x page_size must be below 2^31.");
  check(q.table_stride >= q.columns, "table_stride must be at least columns.");
  check(q.token_stride % 8 == 0 && q.head_stride % 8 == 0 && aligned(q.q),
        "q must be 16-byte aligned, with strides that are multiples of 8.");
  check(q.tokens == 0 || (q.q && q.token_request && q.positions),
        "q, token_request and positions must not be NULL.");
  check(q.tokens == 0 || q.requests == 0 || q.columns == 0 || q.table,
        "table must not be NULL.");
  check(q.tokens <= kIntMax && q.tokens * q.q_heads <= kIntMax, "too many tokens for one call.");
  return {q.q,       q.token_stride, q.head_stride,      q.tokens,
          q.requests, q.table_stride, q.q_heads / c.heads, q.columns,
          q.table,   q.token_request, q.positions};
}

kern::KvSelectArgs select_args(const KvCache& cache, const KvQueries& queries, int n,
                               const Check& check) {
  kern::KvSelectArgs a{};
  a.c = cache_of(cache, check);
  a.q = queries_of(queries, a.c, check);
  check(n >= 1 && n <= kern::kKvMaxBlocks, "n must be in [1, 256].");
  check(a.c.summaries != nullptr, "the cache keeps no summaries.");
  a.n = n;
  return a;
}

kern::KvAttendArgs attend_args(const KvCache& cache, const KvQueries& queries, bool listed, int n,
                               int64_t longest, const Check& check) {
  kern::KvAttendArgs a{};
  a.c = cache_of(cache, check);
  a.q = queries_of(queries, a.c, check);
  check(listed ? n >= 1 && n <= kern::kKvMaxBlocks : n == 0,
        "n must be in [1, 256] with a list of blocks, and 0 without.");
  check(longest >= 0, "longest must not be negative.");
  a.n = n;
  a.longest = longest ? longest : kIntMax;
  kern::kv_attend_plan(a);
  check_grid(kern::kv_attend_grid(a), 256, check);
  return a;
}

}  // namespace

void kv_plan_device(const KvPlan& p, void* stream) {
  const Check check{"mlxvs::kv_plan"};
  const int lps = log2_page(p.page_size, check);
  check(p.requests >= 0 && p.requests <= kIntMax && p.tokens >= 0 && p.tokens <= kIntMax &&
            p.columns >= 0 && p.free_count >= 0 && p.free_count <= kIntMax,
        "requests, columns, free_count and tokens must be in [0, 2^31).");
  check(((int64_t)p.columns << lps) <= kIntMax, "columns x page_size must be below 2^31.");
  check(p.table_stride >= p.columns, "table_stride must be at least columns.");
  check(p.requests == 0 || (p.past && p.fresh && p.lengths && p.first),
        "past, fresh, lengths and first must not be NULL.");
  check(p.requests == 0 || p.columns == 0 || p.table, "table must not be NULL.");
  check(p.free_count == 0 || p.free_pages, "free_pages must not be NULL.");
  check(p.tokens == 0 || (p.slots && p.token_request && p.positions),
        "slots, token_request and positions must not be NULL.");
  check(p.starts && p.cursor && p.cursor_out, "starts, cursor and cursor_out must not be NULL.");
  check(p.cursor != p.cursor_out, "cursor_out must not be cursor.");
  const auto apart = [&](const int32_t* x) {
    return p.lengths + p.requests <= x || x + p.requests <= p.lengths;
  };
  check(p.requests == 0 || (apart(p.past) && apart(p.fresh)),
        "lengths must not overlap past or fresh.");
  check_grid((p.tokens + 255) / 256 + (p.requests + 3) / 4, 256, check);
  detail::need_device();
  const kern::KvPlanArgs a{p.past,      p.fresh,         p.table,     p.free_pages, p.cursor,
                           p.requests,  p.table_stride,  p.free_count, p.tokens,    p.columns,
                           lps,         p.slots,         p.token_request, p.positions, p.starts,
                           p.lengths,   p.first,         p.cursor_out};
  detail::launch_stage<kern::KvPlanArgs, kern::launch_kv_plan>((hipStream_t)stream, "kv_plan", a);
}

void kv_append_device(const KvCache& cache, const void* k, int64_t k_token_stride,
                      int64_t k_head_stride, const void* v, int64_t v_token_stride,
                      int64_t v_head_stride, const int64_t* slots, int64_t tokens, void* stream) {
  const Check check{"mlxvs::kv_append"};
  const kern::KvAppendArgs a{cache_of(cache, check), k, v, k_token_stride, k_head_stride,
                             v_token_stride, v_head_stride, slots, tokens};
  check(tokens >= 0 && tokens <= kIntMax, "tokens must be in [0, 2^31).");
  check(tokens == 0 || (k && v && slots), "k, v and slots must not be NULL.");
  check(aligned(k) && aligned(v) && k_token_stride % 8 == 0 && k_head_stride % 8 == 0 &&
            v_token_stride % 8 == 0 && v_head_stride % 8 == 0,
        "k and v must be 16-byte aligned, with strides that are multiples of 8.");
  check_grid(kern::kv_append_grid(a), 256, check);
  if (tokens == 0) return;
  detail::need_device();
  detail::launch_stage<kern::KvAppendArgs, kern::launch_kv_append>((hipStream_t)stream,
                                                                   "kv_append", a);
}

int64_t kv_select_workspace(const KvCache& cache, const KvQueries& queries, int n) {
  const Check check{"mlxvs::kv_select"};
  return kern::kv_select_workspace(select_args(cache, queries, n, check));
}

void kv_select_device(const KvCache& cache, const KvQueries& queries, int n, int first, int last,
                      int32_t* blocks, void* workspace, int64_t workspace_bytes, void* stream) {
  const Check check{"mlxvs::kv_select"};
  kern::KvSelectArgs a = select_args(cache, queries, n, check);
  check(first >= 0 && last >= 1 && first <= n && last <= n && first + last <= n,
        "first >= 0, last >= 1 and first + last <= n are needed.");
  check(a.q.tokens == 0 || blocks, "blocks must not be NULL.");
  const int64_t need = kern::kv_select_workspace(a);
  check(need == 0 || (workspace && workspace_bytes >= need && aligned(workspace)),
        "the workspace is too small, or not 16-byte aligned.");
  check_grid(kern::kv_select_grid(a), 256, check);
  if (a.q.tokens == 0) return;
  detail::need_device();
  a.first = first;
  a.last = last;
  a.blocks = blocks;
  a.keys = (uint32_t*)workspace;
  detail::launch_stage<kern::KvSelectArgs, kern::launch_kv_select>((hipStream_t)stream,
                                                                   "kv_select", a);
}

int64_t kv_attend_workspace(const KvCache& cache, const KvQueries& queries, int n,
                            int64_t longest) {
  const Check check{"mlxvs::kv_attend"};
  return kern::kv_attend_workspace(attend_args(cache, queries, n != 0, n, longest, check));
}

void kv_attend_device(const KvCache& cache, const KvQueries& queries, const int32_t* blocks, int n,
                      float scale, int64_t longest, void* out, float* lse, void* workspace,
                      int64_t workspace_bytes, void* stream) {
  const Check check{"mlxvs::kv_attend"};
  kern::KvAttendArgs a = attend_args(cache, queries, blocks != nullptr, n, longest, check);
  check(scale > 0.0f && std::isfinite(scale), "scale must be positive and finite.");
  check(a.q.tokens == 0 || out, "out must not be NULL.");
  check(aligned(out), "out must be 16-byte aligned.");
  const int64_t need = kern::kv_attend_workspace(a);
  check(need == 0 || (workspace && workspace_bytes >= need && aligned(workspace)),
        "the workspace is too small, or not 16-byte aligned.");
  if (a.q.tokens == 0) return;
  detail::need_device();
  a.blocks = blocks;
  a.scale = scale;
  a.out = out;
  a.lse = lse;
  a.part_o = (float*)workspace;
  a.part_ml = a.part_o + need / 4 / (a.c.dim + 2) * a.c.dim;
  detail::launch_stage<kern::KvAttendArgs, kern::launch_kv_attend>((hipStream_t)stream,
                                                                   "kv_attend", a);
}

}  // namespace mlxvs
