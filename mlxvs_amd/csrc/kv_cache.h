// Launch interface between the host side (kv_engine.cpp) and the gfx950
// kernels of the paged key-value cache (kv_plan.hip, kv_append.hip,
// kv_select.hip, kv_attend.hip).
//
// Layout, for pages of `page` = 2^lps tokens (16 to 256), `heads` kv heads and
// `dim` values a head (a multiple of 8, at most 256), binary16 or bfloat16:
//   keys      [pages][heads][page][dim]
//   values    [pages][heads][dim][page]   transposed within a page: both MFMA
//             operands that come from the cache then are 16-byte loads of
//             consecutive values straight into registers
//   summaries int8 [pages][heads][dim], scales float32 [pages][heads]
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mlxvs::kern {

constexpr int kKvMaxDim = 256;
constexpr int kKvMaxBlocks = 256;  // entries of a list of selected blocks

struct KvCache {
  void* keys;
  void* values;
  int8_t* summaries;
  float* scales;
  int64_t pages;
  int heads, dim, page, lps;
  int bf16;
};

struct KvPlanArgs {
  const int32_t* past;    // [requests] tokens held before the step
  const int32_t* fresh;   // [requests] tokens of the step
  int32_t* table;         // [requests][cols], rows `table_stride` apart
  const int32_t* free_pages;
  const int32_t* cursor;  // [1]: the first unused entry of free_pages
  int64_t requests, table_stride, free_count, tokens;
  int cols, lps;
  int64_t* slots;         // [tokens]
  int32_t* token_request; // [tokens]
  int32_t* positions;     // [tokens]
  int32_t* starts;        // [requests + 1]
  int32_t* lengths;       // [requests]
  int32_t* first;         // [requests]: a request's first entry of free_pages, -1: not admitted
  int32_t* cursor_out;    // [1]
};
hipError_t launch_kv_plan(const KvPlanArgs& a, hipStream_t s);

struct KvAppendArgs {
  KvCache c;
  const void* k;  // [tokens][heads][dim], token and head strides in values
  const void* v;
  int64_t k_token, k_head, v_token, v_head;
  const int64_t* slots;
  int64_t tokens;
};
int64_t kv_append_grid(const KvAppendArgs& a);  // workgroups of its largest launch
hipError_t launch_kv_append(const KvAppendArgs& a, hipStream_t s);

// Queries of tokens and where they stand.
struct KvQueries {
  const void* q;  // [tokens][heads * group][dim]
  int64_t q_token, q_head;
  int64_t tokens, requests, table_stride;
  int group, cols;
  const int32_t* table;
  const int32_t* token_request;
  const int32_t* positions;
};

struct KvSelectArgs {
  KvCache c;
  KvQueries q;
  int n, first, last;
  int32_t* blocks;  // [tokens][heads][n]
  uint32_t* keys;   // [tokens][heads][cols] ranks, where they do not stay in LDS
};
// Bytes of workspace a call needs (0: none).
int64_t kv_select_workspace(const KvSelectArgs& a);
int64_t kv_select_grid(const KvSelectArgs& a);  // workgroups of its largest launch
hipError_t launch_kv_select(const KvSelectArgs& a, hipStream_t s);

struct KvAttendArgs {
  KvCache c;
  KvQueries q;
  const int32_t* blocks;  // [tokens][heads][n], or null: every block
  int n;                  // entries of a list, 0: every block
  float scale;
  void* out;   // [tokens][heads * group][dim]
  float* lse;  // [tokens][heads * group] or null
  int64_t longest;  // tokens the longest request is expected to hold, INT32_MAX: unknown
  // the split, from kv_attend_plan
  int splits;       // parts of a row's keys, joined by a second launch if more than one
  int chunk;        // keys of a part (a multiple of 64; the last part takes the rest)
  bool shared;      // neighbouring tokens share wavefronts (no parts)
  bool mixed;       // those of prompts do, the others have parts: as the device finds them,
  int span, least;  // by spans of so many tokens, if at least so many are a prompt's
  float* part_o;    // [tokens][heads][group][splits][dim]
  float* part_ml;   // [tokens][heads][group][splits][2]
};
void kv_attend_plan(KvAttendArgs& a);  // sets the split
int64_t kv_attend_workspace(const KvAttendArgs& a);
int64_t kv_attend_grid(const KvAttendArgs& a);  // workgroups of its largest launch
hipError_t launch_kv_attend(const KvAttendArgs& a, hipStream_t s);

}  // namespace mlxvs::kern
