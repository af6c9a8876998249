// Host side of the paged key-value cache: argument checks, the kernels'
// argument blocks, and the C++ API of include/mlxvs/mlxvs.hpp.  The calls
// allocate nothing and keep no state, so unlike the search entries they need no
// per-device lock and no order among themselves.
#include <hip/hip_runtime.h>

#include <algorithm>
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

// (`named`: token_request is read)
kern::KvQueries queries_of(const KvQueries& q, const kern::KvCache& c, const Check& check,
                           bool named = true) {
  check(q.tokens >= 0 && q.requests >= 0 && q.requests <= kIntMax && q.columns >= 0,
        "tokens, requests and columns must not be negative.");
  check(q.q_heads >= c.heads && q.q_heads % c.heads == 0 && q.q_heads <= 1 << 20,
        "q_heads must be a multiple of the cache's heads.");
  check(((int64_t)q.columns << c.lps) <= kIntMax, "columns x page_size must be below 2^31.");
  check(q.table_stride >= q.columns, "table_stride must be at least columns.");
  check(q.token_stride % 8 == 0 && q.head_stride % 8 == 0 && aligned(q.q),
        "q must be 16-byte aligned, with strides that are multiples of 8.");
  check(q.tokens == 0 || (q.q && (q.token_request || !named) && q.positions),
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

kern::KvWeighArgs weigh_args(const KvCache& cache, const KvQueries& queries, int64_t longest,
                             const Check& check) {
  kern::KvWeighArgs a{};
  a.c = cache_of(cache, check);
  a.q = queries_of(queries, a.c, check, false);
  check(longest >= 0, "longest must not be negative.");
  a.longest = longest ? longest : kIntMax;
  kern::kv_weigh_plan(a);
  check_grid(kern::kv_weigh_grid(a), 256, check);
  return a;
}

// Whether [tokens][heads][dim] places with these strides, in values, are apart.
bool apart(int64_t tokens, int64_t token, int64_t heads, int64_t head, int64_t dim) {
  if (tokens <= 1 && heads <= 1) return true;
  if (tokens <= 1) return head >= dim;
  if (heads <= 1) return token >= dim;
  return (head >= dim && token >= (heads - 1) * head + dim) ||
         (token >= dim && head >= (tokens - 1) * token + dim);
}

kern::KvRows rows_of(const KvHeads& x, int64_t tokens, int dim, const Check& check) {
  check(x.heads >= 0 && x.heads <= 1 << 20, "heads must be in [0, 2^20].");
  if (x.heads == 0 || tokens == 0) return {};
  check(x.x && x.out, "rows and their outputs must not be NULL.");
  check(aligned(x.x) && x.token_stride % 8 == 0 && x.head_stride % 8 == 0 && aligned(x.out) &&
            x.out_token_stride % 8 == 0 && x.out_head_stride % 8 == 0 && aligned(x.norm),
        "rows and norms must be 16-byte aligned, with strides that are multiples of 8.");
  check(apart(tokens, x.out_token_stride, x.heads, x.out_head_stride, dim),
        "outputs must not overlap one another.");
  check(x.x != x.out || ((tokens <= 1 || x.token_stride == x.out_token_stride) &&
                         (x.heads <= 1 || x.head_stride == x.out_head_stride)),
        "rows that are written in place must have their own strides.");
  return {x.x,    x.token_stride,          x.head_stride,      x.heads,
          x.norm, x.norm_type == KvNorm::Float32, x.out, x.out_token_stride, x.out_head_stride};
}

kern::KvKeepArgs keep_args(int64_t requests, int32_t heads, int64_t slots, const Check& check) {
  check(requests >= 0 && requests <= kIntMax && heads >= 1 && heads <= 1 << 16 && slots >= 0 &&
            slots <= kIntMax,
        "requests and slots must be in [0, 2^31), heads in [1, 65536].");
  kern::KvKeepArgs a{};
  a.requests = requests;
  a.heads = heads;
  a.slots = slots;
  check_grid(kern::kv_keep_grid(a), 1024, check);
  return a;
}

kern::KvCompactArgs compact_args(const KvCache& cache, const KvCompact& p, const Check& check) {
  kern::KvCompactArgs a{};
  a.c = cache_of(cache, check);
  check(p.requests >= 0 && p.requests <= kIntMax && p.columns >= 0 && p.free_count >= 0 &&
            p.free_count <= kIntMax,
        "requests, columns and free_count must be in [0, 2^31).");
  check(((int64_t)p.columns << a.c.lps) <= kIntMax, "columns x page_size must be below 2^31.");
  check(p.table_stride >= p.columns, "table_stride must be at least columns.");
  check(p.n >= 1, "n must be at least 1.");
  check(p.mass == nullptr || p.slots >= (int64_t)p.columns << a.c.lps,
        "mass must have a slot for each token of the table.");
  a.table = p.table;
  a.table_stride = p.table_stride;
  a.requests = p.requests;
  a.free_count = p.free_count;
  a.cols = p.columns;
  a.n = p.n;
  a.lengths = p.lengths;
  a.kept = p.kept;
  a.free_pages = p.free_pages;
  a.cursor = p.cursor;
  a.mass = p.mass;
  a.slots = p.slots;
  a.lengths_out = p.lengths_out;
  a.cursor_out = p.cursor_out;
  check_grid(kern::kv_compact_grid(a), 256, check);
  return a;
}

}  // namespace

void kv_rotary_frequencies(int32_t rotated, double base, KvScaling scaling, double factor,
                           double context, double* frequencies, float* magnitude) {
  const Check check{"mlxvs::kv_rotary"};
  check(rotated >= 0 && rotated <= kern::kKvMaxDim && rotated % 2 == 0,
        "rotated must be even, in [0, 256].");
  check(base > 1.0 && std::isfinite(base), "base must be finite and greater than 1.");
  check((frequencies || rotated == 0) && magnitude, "frequencies and magnitude must not be NULL.");
  const bool scaled = scaling != KvScaling::None;
  check(!scaled || (factor >= 1.0 && std::isfinite(factor)),
        "factor must be finite and at least 1.");
  check(scaling != KvScaling::Base || rotated > 2, "a scaled base needs more than 2 values.");
  check(scaling != KvScaling::Ramp || (context >= 1.0 && std::isfinite(context)),
        "context must be finite and at least 1.");
  if (scaling == KvScaling::Base) base *= std::pow(factor, (double)rotated / (rotated - 2));
  check(std::isfinite(base), "factor is too large.");
  *magnitude = scaling == KvScaling::Ramp ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
  for (int i = 0; i < rotated / 2; ++i) {
    double f = std::pow(base, -2.0 * i / rotated);
    if (scaling == KvScaling::Linear) f /= factor;
    if (scaling == KvScaling::Ramp) {
      // what turns often within the context stays, what turns less than once is
      // stretched, with a straight line from 32 turns to 1 between them
      const double turns = context * f / (2.0 * M_PI);
      const double stays = std::min(1.0, std::max(0.0, (turns - 1.0) / 31.0));
      f = f * stays + f / factor * (1.0 - stays);
    }
    frequencies[i] = f;
  }
}

void kv_rotary_turns(const double* frequencies, int32_t n, uint64_t* turns) {
  const Check check{"mlxvs::kv_rotary"};
  check(n >= 0 && n <= kern::kKvMaxDim / 2, "n must be in [0, 128].");
  check(n == 0 || (frequencies && turns), "frequencies and turns must not be NULL.");
  for (int i = 0; i < n; ++i) {
    check(std::fabs(frequencies[i]) < 1e6, "frequencies must be finite, below 10^6.");
    const long double t = (long double)frequencies[i] / (2.0L * acosl(-1.0L));
    const long double whole = floorl(t), part = (t - whole) * 0x1p64L;
    turns[i] = part < 0x1p64L ? (uint64_t)part : 0;  // (it may round to a whole turn)
  }
}

void kv_rotate_device(const KvRotary& rotary, const KvHeads& q, const KvHeads& k, int64_t tokens,
                      const int32_t* positions, const int32_t* token_request,
                      const int32_t* evicted, int64_t requests, float eps, void* stream) {
  const Check check{"mlxvs::kv_rotate"};
  check(rotary.dim >= 8 && rotary.dim <= kern::kKvMaxDim && rotary.dim % 8 == 0,
        "dim must be a multiple of 8 in [8, 256].");
  check(rotary.rotated >= 0 && rotary.rotated <= rotary.dim && rotary.rotated % 2 == 0,
        "rotated must be even, in [0, dim].");
  check(rotary.rotated == 0 || rotary.turns, "turns must not be NULL.");
  check(std::isfinite(rotary.magnitude), "magnitude must be finite.");
  check(eps >= 0.0f && std::isfinite(eps), "eps must be finite and not negative.");
  check(tokens >= 0 && tokens <= kIntMax && requests >= 0 && requests <= kIntMax,
        "tokens and requests must be in [0, 2^31).");
  check(tokens == 0 || positions, "positions must not be NULL.");
  check(evicted == nullptr || tokens == 0 || token_request, "evicted needs token_request.");
  kern::KvRotateArgs a{};
  a.q = rows_of(q, tokens, rotary.dim, check);
  a.k = rows_of(k, tokens, rotary.dim, check);
  a.turns = rotary.turns;
  a.dim = rotary.dim;
  a.rotated = rotary.rotated;
  a.pairs = rotary.layout == KvRotaryLayout::Pairs;
  a.bf16 = rotary.type == KvType::BFloat16;
  a.magnitude = rotary.magnitude;
  a.eps = eps;
  a.tokens = tokens;
  a.requests = requests;
  a.positions = positions;
  a.token_request = token_request;
  a.evicted = evicted;
  check_grid(kern::kv_rotate_grid(a), 256, check);
  if (tokens == 0 || a.q.heads + a.k.heads == 0) return;
  detail::need_device();
  detail::launch_stage<kern::KvRotateArgs, kern::launch_kv_rotate>((hipStream_t)stream,
                                                                   "kv_rotate", a);
}

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

int64_t kv_weigh_workspace(const KvCache& cache, const KvQueries& queries, int64_t longest) {
  const Check check{"mlxvs::kv_weigh"};
  return kern::kv_weigh_workspace(weigh_args(cache, queries, longest, check));
}

void kv_weigh_device(const KvCache& cache, const KvQueries& queries, const int32_t* starts,
                     const float* lse, float scale, float decay, int64_t longest, float* mass,
                     int64_t slots, void* workspace, int64_t workspace_bytes, void* stream) {
  const Check check{"mlxvs::kv_weigh"};
  kern::KvWeighArgs a = weigh_args(cache, queries, longest, check);
  check(scale > 0.0f && std::isfinite(scale), "scale must be positive and finite.");
  check(decay >= 0.0f && decay <= 1.0f, "decay must be in [0, 1].");
  check(slots >= (int64_t)a.q.cols << a.c.lps,
        "mass must have a slot for each token of the table.");
  check(a.q.tokens == 0 || a.q.requests == 0 || (starts && lse && mass),
        "starts, lse and mass must not be NULL.");
  const int64_t need = kern::kv_weigh_workspace(a);
  check(need == 0 || (workspace && workspace_bytes >= need && aligned(workspace)),
        "the workspace is too small, or not 16-byte aligned.");
  if (a.q.tokens == 0 || a.q.requests == 0 || a.q.cols == 0) return;
  detail::need_device();
  a.starts = starts;
  a.lse = lse;
  a.scale = scale;
  a.decay = decay;
  a.mass = mass;
  a.slots = slots;
  a.work = (int32_t*)workspace;
  detail::launch_stage<kern::KvWeighArgs, kern::launch_kv_weigh>((hipStream_t)stream, "kv_weigh",
                                                                 a);
}

int64_t kv_keep_workspace(int64_t requests, int32_t heads, int64_t slots) {
  const Check check{"mlxvs::kv_keep"};
  return kern::kv_keep_workspace(keep_args(requests, heads, slots, check));
}

void kv_keep_device(const float* mass, int64_t requests, int32_t heads, int64_t slots,
                    const int32_t* lengths, int32_t n, int32_t first, int32_t recent,
                    int32_t above, int32_t* kept, void* workspace, int64_t workspace_bytes,
                    void* stream) {
  const Check check{"mlxvs::kv_keep"};
  kern::KvKeepArgs a = keep_args(requests, heads, slots, check);
  check(n >= 1, "n must be at least 1.");
  check(first >= 0 && recent >= 0 && first <= n && recent <= n - first,
        "first >= 0, recent >= 0 and first + recent <= n are needed.");
  check(above >= n, "above must be at least n.");
  check(requests == 0 || (lengths && kept && (mass || slots == 0)),
        "mass, lengths and kept must not be NULL.");
  const int64_t need = kern::kv_keep_workspace(a);
  check(need == 0 || (workspace && workspace_bytes >= need && aligned(workspace)),
        "the workspace is too small, or not 16-byte aligned.");
  if (requests == 0) return;
  detail::need_device();
  a.mass = mass;
  a.lengths = lengths;
  a.n = n;
  a.first = first;
  a.recent = recent;
  a.above = above;
  a.kept = kept;
  a.work = workspace;
  detail::launch_stage<kern::KvKeepArgs, kern::launch_kv_keep>((hipStream_t)stream, "kv_keep", a);
}

int64_t kv_compact_workspace(const KvCache& cache, const KvCompact& compact) {
  const Check check{"mlxvs::kv_compact"};
  return kern::kv_compact_workspace(compact_args(cache, compact, check));
}

void kv_compact_device(const KvCache& cache, const KvCompact& p, void* workspace,
                       int64_t workspace_bytes, void* stream) {
  const Check check{"mlxvs::kv_compact"};
  kern::KvCompactArgs a = compact_args(cache, p, check);
  check(p.cursor && p.cursor_out && p.cursor != p.cursor_out,
        "cursor and cursor_out must not be NULL, nor the same.");
  check(p.requests == 0 || (p.lengths && p.lengths_out && p.kept && (p.table || p.columns == 0)),
        "table, lengths, kept and lengths_out must not be NULL.");
  check(p.free_count == 0 || p.free_pages, "free_pages must not be NULL.");
  check(p.requests == 0 || p.lengths_out + p.requests <= p.lengths ||
            p.lengths + p.requests <= p.lengths_out,
        "lengths_out must not overlap lengths.");
  const int64_t need = kern::kv_compact_workspace(a);
  check(need == 0 || (workspace && workspace_bytes >= need && aligned(workspace)),
        "the workspace is too small, or not 16-byte aligned.");
  detail::need_device();
  a.work = (int32_t*)workspace;
  detail::launch_stage<kern::KvCompactArgs, kern::launch_kv_compact>((hipStream_t)stream,
                                                                     "kv_compact", a);
}

}  // namespace mlxvs
