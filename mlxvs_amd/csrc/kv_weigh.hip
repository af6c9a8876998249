// The attention that each cached key gets: for every key p of a request and kv
// head, over the step's tokens t that see it and the head's query heads g,
//
//   mass_p = (p < first ? decay mass_p : 0) + sum_t sum_g exp(scale q_tg.k_p - lse_tg)
//
// with the logarithms of sums that attention over the same keys returned; first is
// the request's first new position, so that a key's mass starts with its own step.
// A key's sum has one owner, or a few whose sums are added in their order: no
// atomics, the same bits every time.
//
// Single tokens read each key once, on the 16x16x32 MFMA with keys straight into
// registers.  Prompts: S = K Q^T on the 32x32x16 MFMA with the keys as rows.  A
// wavefront keeps 64 keys in registers, the operand of every product; the rows of Q
// (a token's query head each) come through LDS by direct loads, whole tokens of up
// to 64 rows at a time, three tiles ahead, for all four wavefronts.  A lane adds up
// its column's weights of each of its 32 keys over all rows, and the 32 columns
// meet once at the end.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "kv_cache.h"
#include "kv_mfma.h"
#include "lds_stage.h"

namespace mlxvs::kern {
namespace {

constexpr int kChunk = 256;  // keys of a workgroup

// x, which is the same in all lanes.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// A request's tokens of the step, and the keys that they see.
struct Span {
  int begin, tokens;
  int first, last;  // positions of the first and the last token
};

__device__ __forceinline__ Span span_of(const KvWeighArgs& a, int64_t r) {
  Span s;
  const int64_t lo = a.starts[r], hi = a.starts[r + 1];
  s.begin = (int)min(max(lo, (int64_t)0), a.q.tokens);
  s.tokens = (int)(min(max(hi, (int64_t)s.begin), a.q.tokens) - s.begin);
  s.first = s.last = -1;
  if (s.tokens > 0) {
    const int end = (a.q.cols << a.c.lps) - 1;
    s.first = a.q.positions[s.begin];
    s.last = min(a.q.positions[s.begin + s.tokens - 1], end);
  }
  return s;
}

// What a key got before, and gets now.
__device__ __forceinline__ void put(const KvWeighArgs& a, float* mass, int p, int first, float got) {
  const float before = p < first && a.decay != 0.0f ? a.decay * mass[p] : 0.0f;
  mass[p] = before + got;
}

// ---- single tokens -------------------------------------------------------------

constexpr int kFewKeys = 16, kFewTiles = 4;  // of a wavefront

// The sum over the 16 lanes of a row.
__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
  for (int i = 8; i >= 1; i >>= 1) x += __shfl_xor(x, i);
  return x;
}

template <int DP, bool BF16>
__global__ __launch_bounds__(256, 2) void kv_weigh_few_kernel(KvWeighArgs a, int chunks) {
  using T = std::conditional_t<BF16, __bf16, _Float16>;
  using Tx8 = std::conditional_t<BF16, bf16x8, halfx8>;
  constexpr int kSteps = DP / 32;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, grp = lane >> 4;
  const int d = a.c.dim, group = a.q.group;
  const int h = (int)(blockIdx.x % a.c.heads);
  const int64_t rest = blockIdx.x / a.c.heads;
  const int r = (int)(rest % a.q.requests);
  const Span sp = span_of(a, r);
  const int32_t* table = a.q.table + (int64_t)r * a.q.table_stride;
  float* mass = a.mass + ((int64_t)r * a.c.heads + h) * a.slots;

  for (int64_t at = rest / a.q.requests * kChunk; at <= sp.last; at += (int64_t)chunks * kChunk) {
    const int k0 = (int)at + wave * (kFewKeys * kFewTiles);
    if (k0 > sp.last) return;
    uintx4 kf[kFewTiles][kSteps];
    bool there[kFewTiles];
#pragma unroll
    for (int u = 0; u < kFewTiles; ++u) {
      const int k = k0 + kFewKeys * u;
      const int page = k <= sp.last ? table[k >> a.c.lps] : -1;
      there[u] = page >= 0 && page < a.c.pages;
      const T* row = (const T*)a.c.keys +
                     (((int64_t)(there[u] ? page : 0) * a.c.heads + h) * a.c.page +
                      ((k & (a.c.page - 1)) + col)) * d + 8 * grp;
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        kf[u][i] = uintx4{};
        if (there[u] && (32 * i + 32 <= sure_values(DP) || 32 * i + 8 * grp < d))
          kf[u][i] = *(const uintx4*)(row + 32 * i);
      }
    }
    float sum[kFewTiles][4] = {};
    const int64_t rows = (int64_t)sp.tokens * group;
    for (int64_t x0 = 0; x0 < rows; x0 += 16) {
      const int64_t x = x0 + col;
      const bool mine = x < rows;
      const int64_t t = sp.begin + (mine ? x / group : 0);
      const int g = h * group + (mine ? (int)(x % group) : 0);
      const int pos = mine ? max(-1, a.q.positions[t]) : -1;
      if (!__any(pos >= k0)) continue;
      const float lse = a.lse[t * a.c.heads * group + g];
      const T* src = (const T*)a.q.q + t * a.q.q_token + g * a.q.q_head + 8 * grp;
      uintx4 q[kSteps];
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        q[i] = uintx4{};
        if (32 * i + 32 <= sure_values(DP) || 32 * i + 8 * grp < d)
          q[i] = *(const uintx4*)(src + 32 * i);
      }
#pragma unroll
      for (int u = 0; u < kFewTiles; ++u) {
        floatx4 s = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
          s = mfma(__builtin_bit_cast(Tx8, kf[u][i]), __builtin_bit_cast(Tx8, q[i]), s);
        const int seen = pos - (k0 + kFewKeys * u + 4 * grp);  // keys up to this one
#pragma unroll
        for (int i = 0; i < 4; ++i)
          sum[u][i] += i <= seen ? __builtin_amdgcn_exp2f(fmaf(s[i], a.scale, -lse) * kLog2e) : 0.0f;
      }
    }
#pragma unroll
    for (int u = 0; u < kFewTiles; ++u) {
      float mine = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float all = row_sum(sum[u][i]);
        if (col == i) mine = all;
      }
      const int p = k0 + kFewKeys * u + 4 * grp + col;
      if (col < 4 && p <= sp.last) put(a, mass, p, sp.first, there[u] ? mine : 0.0f);
    }
  }
}

// ---- prompts -------------------------------------------------------------------

constexpr int kWaveKeys = 64;
constexpr int kRows = 64;    // of a tile of Q
constexpr int kStages = 4;   // tiles in LDS: one in use, the others on their way

// A workgroup's share: a chunk of a request's keys, and some tokens that see it.
struct Unit {
  int request, chunk;
  int begin, end;   // tokens of the batch
  int slot;         // where its sums go, -1: into the masses
  int first, last;  // of the request's positions
  int pieces;       // of the chunk, at its first unit: sums in as many slots
};

// The workspace, made by one workgroup: the units, and those of chunks that several
// units share.
struct Work {
  int32_t* units;   // [1] how many there are, and chunks of several
  int32_t* shared;  // [1]
  int32_t* first;   // [requests + 1] chunks before a request's
  Unit* unit;
  Unit* several;    // the first units of chunks of several
  float* sums;      // [slots][heads][kChunk]
};

// How many there are at most.
struct Most {
  int64_t units, several, slots;
};

int64_t chunks_of(const KvWeighArgs& a) {
  return std::max<int64_t>(1, (((int64_t)a.q.cols << a.c.lps) + kChunk - 1) / kChunk);
}
__host__ __device__ __forceinline__ int64_t header_ints(const KvWeighArgs& a) {
  return (2 + a.q.requests + 1 + 3) / 4 * 4;
}
__device__ __forceinline__ Work work_of(const KvWeighArgs& a) {
  int32_t* w = a.work;
  Unit* unit = (Unit*)(w + header_ints(a));
  return {w, w + 1, w + 2, unit, unit + a.most_units, (float*)(unit + a.most_units + a.most_several)};
}

constexpr int kPlanThreads = 1024;

// Sums over a workgroup's threads of N numbers up to each; `all` gets the totals.
template <int N>
__device__ __forceinline__ void running(int64_t (&x)[N], int64_t (&all)[N],
                                        int64_t (*waves)[N]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int i = 0; i < N; ++i) {
#pragma unroll
    for (int by = 1; by < 64; by <<= 1) {
      const int64_t y = __shfl_up(x[i], by);
      if (lane >= by) x[i] += y;
    }
    if (lane == 63) waves[wave][i] = x[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    all[i] = 0;
    for (int w = 0; w < kPlanThreads / 64; ++w) {
      if (w < wave) x[i] += waves[w][i];
      all[i] += waves[w][i];
    }
  }
  __syncthreads();
}

// The first of a request's tokens whose position is at least p: positions ascend, and
// mostly by one.
__device__ __forceinline__ int first_at(const int32_t* positions, const Span& sp, int p) {
  if (p <= sp.first) return 0;
  int lo = 0, hi = sp.tokens;  // (positions[lo] < p; the answer is in (lo, hi])
  const int guess = min(hi, p - sp.first);
  if (positions[guess - 1] < p) {
    lo = guess - 1;
    if (guess < hi && positions[guess] >= p) return guess;
  } else {
    hi = guess - 1;
  }
  while (hi - lo > 1) {
    const int mid = lo + (hi - lo) / 2;
    if (positions[mid] < p) lo = mid;
    else hi = mid;
  }
  return hi;
}

__global__ __launch_bounds__(kPlanThreads) void kv_weigh_plan_kernel(KvWeighArgs a) {
  __shared__ int64_t waves[kPlanThreads / 64][3];
  const Work work = work_of(a);
  // the requests' chunks ...
  int64_t chunks = 0;
  for (int64_t r0 = 0; r0 < a.q.requests; r0 += kPlanThreads) {
    const int64_t r = r0 + threadIdx.x;
    int64_t n[1] = {0}, all[1];
    if (r < a.q.requests) {
      const Span sp = span_of(a, r);
      n[0] = sp.last < 0 ? 0 : sp.last / kChunk + 1;
    }
    running<1>(n, all, (int64_t(*)[1])waves);
    if (r < a.q.requests) work.first[r + 1] = (int32_t)(chunks + n[0]);
    chunks += all[0];
  }
  if (threadIdx.x == 0) work.first[0] = 0;
  __syncthreads();
  // ... and each one's units
  int64_t before[3] = {0, 0, 0};  // units, chunks of several, slots
  for (int64_t i0 = 0; i0 < chunks; i0 += kPlanThreads) {
    const int64_t i = i0 + threadIdx.x;
    Unit u{};
    Span sp{};
    int from = 0, pieces = 0;
    if (i < chunks) {
      int64_t lo = 0, hi = a.q.requests;  // first[lo] <= i < first[hi]
      while (hi - lo > 1) {
        const int64_t mid = lo + (hi - lo) / 2;
        if (work.first[mid] <= i) lo = mid;
        else hi = mid;
      }
      sp = span_of(a, lo);
      u.request = (int)lo;
      u.chunk = (int)(i - work.first[lo]);
      u.first = sp.first;
      u.last = sp.last;
      from = min(first_at(a.q.positions + sp.begin, sp, u.chunk * kChunk), sp.tokens - 1);
      pieces = (int)((sp.tokens - from + a.piece - 1) / a.piece);
      u.pieces = pieces;
    }
    int64_t x[3] = {pieces, pieces > 1, pieces > 1 ? pieces : 0}, all[3];
    const int64_t own[3] = {x[0], x[1], x[2]};
    running<3>(x, all, waves);
    if (i < chunks) {
      const int64_t at = before[0] + x[0] - own[0], slot = before[2] + x[2] - own[2];
      // (all of a chunk's units have as many tiles, or one less)
      const int tokens = sp.tokens - from, each = max(1, kRows / a.q.group);
      const int tiles = (tokens + each - 1) / each;
      for (int p = 0; p < pieces; ++p) {
        u.begin = sp.begin + from + (int)((int64_t)tiles * p / pieces) * each;
        u.end = sp.begin + min(sp.tokens, from + (int)((int64_t)tiles * (p + 1) / pieces) * each);
        u.slot = pieces > 1 ? (int)(slot + p) : -1;
        work.unit[at + p] = u;
        if (p == 0 && pieces > 1) work.several[before[1] + x[1] - 1] = u;
      }
    }
#pragma unroll
    for (int j = 0; j < 3; ++j) before[j] += all[j];
  }
  if (threadIdx.x == 0) {
    work.units[0] = (int32_t)before[0];
    work.shared[0] = (int32_t)before[1];
  }
}

// What rows of a tile have past the head.  Rows that no token fills are zeros with a
// logarithm that leaves no weight, and see all keys, so that a tile of them takes
// the short way; rows that are not the unit's see none.
__device__ const uintx4 kZeros = {};
__device__ const float kNoLse = __builtin_inff();
__device__ const int kNoRowsPosition = INT32_MAX, kNoPosition = -1;

// DP: head size rounded up.
template <int DP, bool BF16>
struct Weigh {
  using T = std::conditional_t<BF16, __bf16, _Float16>;
  using Tx8 = std::conditional_t<BF16, bf16x8, halfx8>;
  static constexpr int kSteps = DP / 16;
  // A tile in LDS: rows of 16-byte chunks, their logarithms and positions, and
  // 256 bytes that are not read.  A chunk's place in its row is swapped so that 16
  // rows' same chunk lies in all banks; tiles are aligned so that it is some bits of
  // its address.
  static constexpr int kRow = DP <= 64 ? 8 : DP <= 128 ? 16 : 32;
  static constexpr int kLse = kRows * kRow * 16, kPos = kLse + 4 * kRows, kNone = kPos + 4 * kRows;
  static constexpr int kTileBytes = (kNone + 4 * kRows + 511) / 512 * 512;
  static constexpr int kCopies = kRow / 4;  // of 1 KB a wavefront and tile
  static constexpr int kLoads = kCopies + 1;  // ... and one of 256 bytes
  __device__ __forceinline__ static int swap(int row) {
    return kRow == 8 ? row >> 1 & 7 : row & 15;
  }

  const KvWeighArgs& a;
  const int lane, wave, h, group;
  const int heads_tile, tokens_tile;  // a tile: heads of a token, or all of some tokens
  const bool gaps;        // it has chunks or rows that are zeros
  int64_t rows[kCopies];  // this lane's pieces of a tile, from its first row on
  static constexpr int64_t kNoRow = INT64_MIN;
  int token_told, head_told;  // the row whose logarithm or position it brings; -1: none
  int told;                   // ... from the tile's first row on
  int token, end, head;   // the next tile's first, one past the last of all, its head
  uintx4 kf[2][kSteps];
  float sum[32];

  __device__ __forceinline__ Weigh(const KvWeighArgs& args, int hd)
      : a(args), lane(threadIdx.x & 63), wave(uniform(threadIdx.x >> 6)), h(hd), group(args.q.group),
        heads_tile(min(args.q.group, kRows)), tokens_tile(max(1, kRows / args.q.group)),
        gaps(args.c.dim != 8 * kRow || heads_tile * tokens_tile != kRows) {
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int slot = (wave + 4 * i) * 64 + lane, j = slot / kRow, chunk = (slot % kRow) ^ swap(j);
      // (tokens past the batch's: another one)
      const int t = min(j / heads_tile, (int)a.q.tokens - 1);
      rows[i] = t * a.q.q_token + j % heads_tile * a.q.q_head + 8 * chunk;
      if (8 * chunk >= a.c.dim || j / heads_tile >= tokens_tile) rows[i] = kNoRow;
    }
    token_told = lane / heads_tile < tokens_tile ? lane / heads_tile : -1;
    head_told = lane % heads_tile;
    told = wave == 0 ? token_told * a.c.heads * group + head_told : token_told;
  }

  // Tokens t0 .. t1 - 1 of the batch; returns their tiles.
  __device__ __forceinline__ int start(int t0, int t1) {
    token = t0;
    end = t1;
    head = 0;
#pragma unroll
    for (int e = 0; e < 32; ++e) sum[e] = 0.0f;
    return (t1 - t0 + tokens_tile - 1) / tokens_tile * ((group + kRows - 1) / kRows);
  }

  // Copies the next tile into LDS (past the last: anything), kLoads loads.  A tile
  // that would reach past the batch, or the group, begins before its first row:
  // rows that are not its own are copied and not seen.
  __device__ __forceinline__ void copy(uint32_t tile) {
    const int t = max(0, min(token, (int)a.q.tokens - tokens_tile)), g = min(head, group - heads_tile);
    const T* q = (const T*)a.q.q + t * a.q.q_token + (int64_t)(h * group + g) * a.q.q_head;
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const void* src = q + rows[i];
      if (gaps && rows[i] == kNoRow) src = &kZeros;
      stream16_to_lds(src, tile + 1024 * (wave + 4 * i));
    }
    // two wavefronts bring what the columns need, the others as much of nothing, so
    // that all have as many loads on their way
    const void* src = &kZeros;
    if (wave < 2) {
      const int x = t + token_told;
      const bool own = token_told >= 0 && x >= token && x < end && g + head_told >= head;
      if (wave == 0) {
        const float* lse = a.lse + ((int64_t)t * a.c.heads + h) * group + g;
        src = own ? lse + told : &kNoLse;
      } else {
        src = own ? a.q.positions + t + told : token_told < 0 ? &kNoRowsPosition : &kNoPosition;
      }
    }
    stream4_to_lds(src, tile + (wave == 0 ? kLse : wave == 1 ? kPos : kNone));
    head += kRows;
    if (head >= group) {
      head = 0;
      token = min(token + tokens_tile, end);
    }
  }

  // The keys k0 .. k0 + 63 of a table's row, zeros where none is.
  __device__ __forceinline__ void keys(const int32_t* table, int k0, int upto) {
    const int d = a.c.dim, col = lane & 31, half = lane >> 5;
    int page[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int k = k0 + 32 * u + col;
      page[u] = k <= upto ? table[k >> a.c.lps] : -1;
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int k = k0 + 32 * u + col;
      const bool there = page[u] >= 0 && page[u] < a.c.pages;
      const T* src = (const T*)a.c.keys +
                     (((int64_t)(there ? page[u] : 0) * a.c.heads + h) * a.c.page +
                      (k & (a.c.page - 1))) * d;
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const int at = 16 * i + 8 * half;
        kf[u][i] = uintx4{};
        if (there && (16 * i + 16 <= sure_values(DP) || at < d)) kf[u][i] = *(const uintx4*)(src + at);
      }
    }
  }

  // The products of 32 rows of a tile.  beside(i) is done while step i's products are
  // made.
  template <bool MIX, typename Beside>
  __device__ __forceinline__ void products(uint32_t tile, int ct, floatx16 (&s)[2], Beside beside) {
    constexpr int kAhead = 4;  // reads of Q
    const int col = lane & 31, half = lane >> 5;
    const uint32_t at = tile + (32 * ct + col) * kRow * 16 + 16 * (half ^ swap(32 * ct + col));
    uintx4 q[kSteps];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) q[i] = lds_read16(at ^ (32 * i));
    s[0] = s[1] = floatx16{};
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      if (i + kAhead < kSteps) q[i + kAhead] = lds_read16(at ^ (32 * (i + kAhead)));
#pragma unroll
      for (int u = 0; u < 2; ++u)
        s[u] = mfma(__builtin_bit_cast(Tx8, kf[u][i]), __builtin_bit_cast(Tx8, q[i]), s[u]);
      beside(i);
      if constexpr (MIX) __builtin_amdgcn_sched_barrier(0);
    }
  }

  // Adds the weights of the keys of a column that belong to step i, all of which it
  // sees.  (The sums are tied to their place: they would be moved behind all
  // products, which then have nothing beside them.)
  __device__ __forceinline__ void add(const floatx16 (&s)[2], int i, float c, float lse) {
    constexpr int kPer = (32 + kSteps - 1) / kSteps;
#pragma unroll
    for (int e = i * kPer; e < (i + 1) * kPer; ++e) {
      if (e >= 32) continue;
      sum[e] += __builtin_amdgcn_exp2f(fmaf(s[e / 16][e % 16], c, -lse));
#if defined(__HIP_DEVICE_COMPILE__)
      asm volatile("" : "+v"(sum[e]));
#endif
    }
  }

  // What a tile's columns are: rows 0 .. 31 and 32 .. 63.
  struct Columns {
    float lse[2];  // times log2(e)
    int pos[2];
  };
  __device__ __forceinline__ Columns columns(uint32_t tile) const {
    const int col = 4 * (lane & 31);
    Columns n;
#pragma unroll
    for (int ct = 0; ct < 2; ++ct) {
      n.lse[ct] = lds_read4<float>(tile + kLse + 128 * ct + col) * kLog2e;
      n.pos[ct] = lds_read4<int>(tile + kPos + 128 * ct + col);
    }
    return n;
  }
  // Whether all of them see all of this wavefront's keys, from k0 on.
  __device__ __forceinline__ bool full(const Columns& n, int k0) const {
    return __all(min(n.pos[0], n.pos[1]) >= k0 + kWaveKeys - 1);
  }

  // A tile of which some see some.
  __device__ __forceinline__ void use_some(uint32_t tile, const Columns& n, int k0, float c) {
#pragma unroll 1
    for (int ct = 0; ct < 2; ++ct) {
      const float lse = ct ? n.lse[1] : n.lse[0];
      const int pos = max(-1, ct ? n.pos[1] : n.pos[0]), seen = pos - k0 - 4 * (lane >> 5);
      if (!__any(pos >= k0)) continue;
      floatx16 s[2];
      products<false>(tile, ct, s, [](int) {});
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        const float x = __builtin_amdgcn_exp2f(fmaf(s[e / 16][e % 16], c, -lse));
        sum[e] += 32 * (e / 16) + 8 * (e % 16 / 4) + e % 4 <= seen ? x : 0.0f;
      }
    }
  }

  // All `todo` tiles against the keys from k0 on; tile(n) is the n-th's place,
  // enter(n) waits for it.
  template <typename Tile, typename Enter>
  __device__ __forceinline__ void run(int todo, int k0, float c, Tile tile, Enter enter) {
    int n = 0;
    while (n < todo) {
      enter(n);
      Columns x = columns(tile(n));
      if (full(x, k0)) {
        // the weights of a half tile are taken while the next one's products are made
        floatx16 open[2] = {};
        float lse = __builtin_inff();
#pragma unroll 1
        while (true) {
          floatx16 s[2];
          products<true>(tile(n), 0, s, [&](int i) { add(open, i, c, lse); });
          products<true>(tile(n), 1, open, [&](int i) { add(s, i, c, x.lse[0]); });
          lse = x.lse[1];
          if (++n == todo) break;
          enter(n);
          x = columns(tile(n));
          if (!full(x, k0)) break;
        }
#pragma unroll
        for (int i = 0; i < kSteps; ++i) add(open, i, c, lse);
        if (n == todo) return;
      }
      use_some(tile(n), x, k0, c);
      ++n;
    }
  }

  // The sums over the columns: lane l's key is key_of(l).
  __device__ __forceinline__ float meet() {
#pragma unroll
    for (int b = 16; b >= 1; b >>= 1)
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        if (j >= b) continue;
        const bool up = lane & b;
        const float mine = up ? sum[j + b] : sum[j], other = up ? sum[j] : sum[j + b];
        sum[j] = mine + __shfl_xor(other, b);
      }
    return sum[0];
  }
  __device__ __forceinline__ static int key_of(int lane) {
    const int e = lane & 31;
    return 32 * (e / 16) + 8 * (e % 16 / 4) + 4 * (lane >> 5) + e % 4;
  }
};

template <int DP, bool BF16>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void kv_weigh_kernel(KvWeighArgs a) {
  using W = Weigh<DP, BF16>;
  __shared__ __align__(512) char tiles[kStages * W::kTileBytes];
  const uint32_t at = lds_address(tiles);
  const Work work = work_of(a);
  const int h = (int)(blockIdx.x % a.c.heads), lane = threadIdx.x & 63;
  const int units = uniform(work.units[0]);
  const float c = a.scale * kLog2e;
  W w(a, h);
  for (int x = (int)(blockIdx.x / a.c.heads); x < units; x += (int)(gridDim.x / a.c.heads)) {
    const Unit u = work.unit[x];
    const int r = uniform(u.request), last = uniform(u.last), slot = uniform(u.slot);
    const int k0 = uniform(u.chunk) * kChunk + w.wave * kWaveKeys;
    const int32_t* table = a.q.table + r * a.q.table_stride;
    const int todo = w.start(uniform(u.begin), uniform(u.end));
#pragma unroll
    for (int n = 0; n < kStages - 1; ++n) w.copy(at + n * W::kTileBytes);
    w.keys(table, k0, last);
    // (known to the compiler, which else waits for the keys, and with them for all
    // that was loaded since, in every turn)
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    const auto tile = [&](int n) { return at + n % kStages * W::kTileBytes; };
    const auto enter = [&](int n) {
      staged_barrier<(kStages - 2) * W::kLoads>();
      mfma_settle();
      w.copy(tile(n + kStages - 1));  // (the place of the one before)
    };
    if (k0 <= last) {
      w.run(todo, k0, c, tile, enter);
    } else {
#pragma unroll 1
      for (int n = 0; n < todo; ++n) enter(n);
    }
    dma_barrier();  // (nothing is on its way into the tiles any more)
    mfma_settle();
    const float got = w.meet();
    const int key = W::key_of(lane), p = k0 + key;
    if (p > last) continue;
    if (slot >= 0) {
      work.sums[((int64_t)slot * a.c.heads + h) * kChunk + w.wave * kWaveKeys + key] = got;
    } else {
      const int page = table[p >> a.c.lps];
      put(a, a.mass + ((int64_t)r * a.c.heads + h) * a.slots, p, u.first,
          page >= 0 && page < a.c.pages ? got : 0.0f);
    }
  }
}

// Adds up the units' sums of a chunk, in their order.
__global__ __launch_bounds__(kChunk) void kv_weigh_join_kernel(KvWeighArgs a) {
  const Work work = work_of(a);
  const int h = (int)(blockIdx.x % a.c.heads), shared = work.shared[0];
  for (int64_t x = blockIdx.x / a.c.heads; x < shared; x += gridDim.x / a.c.heads) {
    const Unit u = work.several[x];
    const int p = u.chunk * kChunk + threadIdx.x;
    if (p > u.last) continue;
    const float* sums = work.sums + ((int64_t)u.slot * a.c.heads + h) * kChunk + threadIdx.x;
    float got = 0.0f;
#pragma unroll 4
    for (int i = 0; i < u.pieces; ++i) got += sums[(int64_t)i * a.c.heads * kChunk];
    const int page = a.q.table[u.request * a.q.table_stride + (p >> a.c.lps)];
    put(a, a.mass + ((int64_t)u.request * a.c.heads + h) * a.slots, p, u.first,
        page >= 0 && page < a.c.pages ? got : 0.0f);
  }
}

// ---- which one ------------------------------------------------------------------

// Workgroups that single tokens' chunks are dealt to, for each request.
int64_t few_chunks(const KvWeighArgs& a) {
  const int64_t most = std::min<int64_t>(a.longest, (int64_t)a.q.cols << a.c.lps);
  return std::max<int64_t>(1, (most + kChunk - 1) / kChunk);
}

constexpr int64_t kGrid = 2048;  // workgroups at most
constexpr int64_t kUnits = 2048;
constexpr int64_t kLeast = 1024;  // rows of a unit

template <int DP, bool BF16>
void launch_dim(const KvWeighArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)kv_weigh_grid(a));
  if (a.piece) kv_weigh_kernel<DP, BF16><<<grid, 256, 0, s>>>(a);
  else kv_weigh_few_kernel<DP, BF16><<<grid, 256, 0, s>>>(a, (int)few_chunks(a));
}

template <bool BF16>
void launch_type(const KvWeighArgs& a, hipStream_t s) {
  if (a.c.dim <= 64) launch_dim<64, BF16>(a, s);
  else if (a.c.dim <= 96) launch_dim<96, BF16>(a, s);
  else if (a.c.dim <= 128) launch_dim<128, BF16>(a, s);
  else if (a.c.dim <= 192) launch_dim<192, BF16>(a, s);
  else launch_dim<256, BF16>(a, s);
}

}  // namespace

void kv_weigh_plan(KvWeighArgs& a) {
  a.piece = a.most_units = a.most_several = a.most_slots = 0;
  if (a.q.tokens <= a.q.requests || a.q.cols == 0) return;
  const int64_t chunks = few_chunks(a), pieces = std::max<int64_t>(1, kUnits / (chunks * a.c.heads));
  const int64_t each = std::max<int64_t>(1, kRows / a.q.group);  // tokens of a tile
  const int64_t piece = std::max((a.q.tokens + pieces - 1) / pieces, kLeast / a.q.group);
  a.piece = (piece + each - 1) / each * each;
  // a chunk of a request of t tokens has at most 1 + t / piece units
  const int64_t all = chunks_of(a), full = a.q.tokens / a.piece;
  a.most_units = all * (a.q.requests + full);
  a.most_several = all * std::min(a.q.requests, full);
  a.most_slots = 2 * all * full;
}

int64_t kv_weigh_workspace(const KvWeighArgs& a) {
  if (!a.piece) return 0;
  return 4 * header_ints(a) + (a.most_units + a.most_several) * (int64_t)sizeof(Unit) +
         a.most_slots * a.c.heads * kChunk * 4;
}

int64_t kv_weigh_grid(const KvWeighArgs& a) {
  if (!a.piece) return a.q.requests * a.c.heads * few_chunks(a);
  return std::min(a.most_units, std::max<int64_t>(1, kGrid / a.c.heads)) * a.c.heads;
}

hipError_t launch_kv_weigh(const KvWeighArgs& a, hipStream_t s) {
  if (a.piece) {
    kv_weigh_plan_kernel<<<1, kPlanThreads, 0, s>>>(a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  a.c.bf16 ? launch_type<true>(a, s) : launch_type<false>(a, s);
  if (hipError_t e = hipGetLastError(); e != hipSuccess || a.most_several == 0) return e;
  const int64_t grid = std::min(a.most_several, std::max<int64_t>(1, kGrid / a.c.heads)) * a.c.heads;
  kv_weigh_join_kernel<<<dim3((unsigned)grid), kChunk, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace mlxvs::kern
