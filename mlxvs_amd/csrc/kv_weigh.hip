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
// S = K Q^T on the 32x32x16 MFMA with the keys as rows.  A wavefront keeps 64 keys
// in registers, the operand of every product; the rows of Q (a token's query
// head each) come through LDS by direct loads, whole tokens of up to 64 rows at a
// time, three tiles ahead, for all four wavefronts.  A lane adds up its column's weights of each of its 32 keys
// over all rows, and the 32 columns meet once at the end.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "kv_cache.h"
#include "kv_mfma.h"
#include "lds_stage.h"

namespace mlxvs::kern {
namespace {

constexpr int kWaveKeys = 64;
constexpr int kChunk = 4 * kWaveKeys;  // keys of a workgroup
constexpr int kRows = 64;              // of a tile of Q

// Prompts are split into pieces of rows where a request's keys alone do not fill
// the card.  The workspace: each request's first piece and, for those of several,
// its first partial sum; which these are; the sums.
struct Work {
  int32_t* count;   // [1] requests of several pieces
  int32_t* first;   // [requests + 1] pieces before a request's
  int32_t* base;    // [requests] partial sums before it, -1: it has one piece
  int32_t* several; // [requests]
  float* sums;      // [partial sums][heads][cols x page]
};

__host__ __device__ __forceinline__ int64_t header_ints(const KvWeighArgs& a) {
  return (1 + a.q.requests + 1 + 2 * a.q.requests + 3) / 4 * 4;
}
__device__ __forceinline__ Work work_of(const KvWeighArgs& a) {
  int32_t* w = a.work;
  return {w, w + 1, w + 2 + a.q.requests, w + 2 + 2 * a.q.requests, (float*)(w + header_ints(a))};
}

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

__device__ __forceinline__ int64_t pieces_of(const KvWeighArgs& a, int tokens) {
  return max((int64_t)1, (tokens + a.piece - 1) / a.piece);
}

constexpr int kPlanThreads = 1024;

__global__ __launch_bounds__(kPlanThreads) void kv_weigh_plan_kernel(KvWeighArgs a) {
  __shared__ int64_t waves[kPlanThreads / 64][3];
  const Work work = work_of(a);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t before[3] = {0, 0, 0};
  for (int64_t r0 = 0; r0 < a.q.requests; r0 += kPlanThreads) {
    const int64_t r = r0 + threadIdx.x;
    int64_t own[3] = {0, 0, 0};  // pieces, partial sums, requests of several
    if (r < a.q.requests) {
      own[0] = pieces_of(a, span_of(a, r).tokens);
      own[1] = own[0] > 1 ? own[0] : 0;
      own[2] = own[0] > 1;
    }
    int64_t upto[3] = {own[0], own[1], own[2]};
#pragma unroll
    for (int x = 0; x < 3; ++x) {
#pragma unroll
      for (int by = 1; by < 64; by <<= 1) {
        const int64_t y = __shfl_up(upto[x], by);
        if (lane >= by) upto[x] += y;
      }
      if (lane == 63) waves[wave][x] = upto[x];
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < 3; ++x) {
      upto[x] += before[x];
      for (int w = 0; w < kPlanThreads / 64; ++w) {
        if (w < wave) upto[x] += waves[w][x];
        before[x] += waves[w][x];
      }
    }
    __syncthreads();
    if (r < a.q.requests) {
      work.first[r] = (int32_t)(upto[0] - own[0]);
      work.base[r] = own[1] ? (int32_t)(upto[1] - own[1]) : -1;
      if (own[2]) work.several[upto[2] - 1] = (int32_t)r;
    }
  }
  if (threadIdx.x == 0) {
    work.first[a.q.requests] = (int32_t)before[0];
    work.count[0] = (int32_t)before[2];
  }
}

// Of n ascending numbers at(0) .. at(n - 1), how many are below x, by a wavefront.
template <typename At>
__device__ __forceinline__ int below(int n, int lane, At at, int x) {
  int lo = 0, hi = n;  // the answer is in [lo, hi]
  while (lo < hi) {
    const int step = (hi - lo + 63) / 64;
    const int i = lo + lane * step;
    const int some = (int)__popcll(__ballot(i < hi && at(i) < x));
    // the last of those is at lo + (some - 1) step; the next one is not below x
    const int next = min(hi, lo + some * step);
    lo = some ? lo + (some - 1) * step + 1 : lo;
    hi = max(lo, next);
  }
  return lo;
}

// What a key got before, and gets now.
__device__ __forceinline__ void put(const KvWeighArgs& a, float* mass, int p, int first, float got) {
  const float before = p < first && a.decay != 0.0f ? a.decay * mass[p] : 0.0f;
  mass[p] = before + got;
}

// What rows of a tile have past the head.  Rows that no token fills are zeros with a
// logarithm that leaves no weight, and see all keys, so that a tile of them takes
// the short way; rows that are not the piece's see none.
__device__ const uintx4 kZeros = {};
__device__ const float kNoLse = __builtin_inff();
__device__ const int kNoRowsPosition = INT32_MAX, kNoPosition = -1;

// x, which is the same in all lanes.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

constexpr int kStages = 4;  // tiles in LDS: one in use, the others on their way

// DP: head size rounded up.
template <int DP, bool BF16>
struct Weigh {
  using T = std::conditional_t<BF16, __bf16, _Float16>;
  using Tx8 = std::conditional_t<BF16, bf16x8, halfx8>;
  static constexpr int kSteps = DP / 16;
  // 16-byte chunks of a row in LDS.  A chunk's place in its row is swapped so that 16
  // rows' same chunk lies in all banks.
  static constexpr int kRow = DP <= 64 ? 8 : DP <= 128 ? 16 : 32;
  static constexpr int kTileBytes = kRows * kRow * 16;
  static constexpr int kCopies = kRow / 4;  // of 1 KB a wavefront and tile
  static constexpr int kLoads = kCopies + 1;  // ... and one of 256 bytes
  __device__ __forceinline__ static int swap(int row) {
    return kRow == 8 ? row >> 1 & 7 : row & 15;
  }

  // (aligned so that a chunk's place in its row is some bits of its address)
  struct __align__(512) Tile {
    char q[kTileBytes];
    float lse[kRows];  // infinity for a row that is not there
    int pos[kRows];
    int none[kRows];
  };

  const KvWeighArgs& a;
  const int lane, wave, h, group;
  const int heads_tile, tokens_tile;  // a tile: heads of a token, or all of some tokens
  int64_t rows[kCopies];  // this lane's pieces of a tile, from its first row on
  int token_told, head_told;  // the row whose logarithm or position it brings; -1: none
  int token, end, head;   // the next tile's first, one past the last of all, its head
  uintx4 kf[2][kSteps];
  float sum[32];

  __device__ __forceinline__ Weigh(const KvWeighArgs& args, int hd)
      : a(args), lane(threadIdx.x & 63), wave(uniform(threadIdx.x >> 6)), h(hd), group(args.q.group),
        heads_tile(min(args.q.group, kRows)), tokens_tile(max(1, kRows / args.q.group)) {
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
  }
  static constexpr int64_t kNoRow = INT64_MIN;

  // Tokens t0 .. t1 - 1 of the batch.
  __device__ __forceinline__ void start(int t0, int t1) {
    token = t0;
    end = t1;
    head = 0;
  }
  __device__ __forceinline__ int tiles() const {
    return (end - token + tokens_tile - 1) / tokens_tile * ((group + kRows - 1) / kRows);
  }

  // Copies the next tile into LDS (past the last: anything), kLoads loads.  A tile
  // that would reach past the batch, or the group, begins before its first row:
  // rows that are not its own are copied and not seen.
  __device__ __forceinline__ void copy(Tile& to) {
    const int t = max(0, min(token, (int)a.q.tokens - tokens_tile)), g = min(head, group - heads_tile);
    const T* q = (const T*)a.q.q + t * a.q.q_token + (int64_t)(h * group + g) * a.q.q_head;
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const void* src = q + rows[i];
      if (rows[i] == kNoRow) src = &kZeros;
      stream16_to_lds(src, to.q + 1024 * (wave + 4 * i));
    }
    // two wavefronts bring what the columns need, the others as much of nothing, so
    // that all have as many loads on their way
    const void* src = &kZeros;
    void* dst = to.none;
    if (wave < 2) {
      const int x = t + token_told;
      const bool own = token_told >= 0 && x >= token && x < end && g + head_told >= head;
      if (wave == 0) {
        src = own ? (const void*)(a.lse + ((int64_t)x * a.c.heads + h) * group + g + head_told) : &kNoLse;
        dst = to.lse;
      } else {
        src = own ? a.q.positions + x : token_told < 0 ? &kNoRowsPosition : &kNoPosition;
        dst = to.pos;
      }
    }
    stream4_to_lds(src, dst);
    head += kRows;
    if (head >= group) {
      head = 0;
      token = min(token + tokens_tile, end);
    }
  }

  // The keys k0 .. k0 + 63 of a table's row, zeros where none is.
  __device__ __forceinline__ void keys(const int32_t* table, int k0, int upto) {
    const int d = a.c.dim, col = lane & 31, half = lane >> 5;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int k = k0 + 32 * u + col;
      const int page = k <= upto ? table[k >> a.c.lps] : -1;
      const bool there = page >= 0 && page < a.c.pages;
      const T* src = (const T*)a.c.keys +
                     (((int64_t)(there ? page : 0) * a.c.heads + h) * a.c.page +
                      (k & (a.c.page - 1))) * d;
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const int at = 16 * i + 8 * half;
        kf[u][i] = uintx4{};
        if (there && (16 * i + 16 <= sure_values(DP) || at < d)) kf[u][i] = *(const uintx4*)(src + at);
      }
    }
  }

  // The products of 32 rows of a tile; between(i) is done beside step i's.
  template <typename Between>
  __device__ __forceinline__ void products(const Tile& tile, int ct, floatx16 (&s)[2],
                                           Between between) const {
    const int col = lane & 31, half = lane >> 5;
    const uint32_t at = lds_address(tile.q) + (32 * ct + col) * kRow * 16 +
                        16 * (half ^ swap(32 * ct + col));
    uintx4 q[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) q[i] = lds_read16(at ^ (32 * i));
#pragma unroll
    for (int u = 0; u < 2; ++u) s[u] = floatx16{};
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
        s[u] = mfma(__builtin_bit_cast(Tx8, kf[u][i]), __builtin_bit_cast(Tx8, q[i]), s[u]);
      between(i);
    }
  }

  // Adds the weights of a column's keys e0 .. e1 - 1, all of which it sees.
  __device__ __forceinline__ void add(const floatx16 (&s)[2], int e0, int e1, float c, float lse) {
#pragma unroll
    for (int e = 0; e < 32; ++e)
      if (e >= e0 && e < e1)
        sum[e] += __builtin_amdgcn_exp2f(fmaf(s[e / 16][e % 16], c, -lse));
  }

  // A tile's rows against this wavefront's keys.
  __device__ __forceinline__ void use(const Tile& tile, int k0, float c) {
    const int col = lane & 31, half = lane >> 5;
    const float l0 = tile.lse[col] * kLog2e, l1 = tile.lse[32 + col] * kLog2e;
    const int p0 = tile.pos[col], p1 = tile.pos[32 + col];
    floatx16 s0[2], s1[2];
    if (__all(min(p0, p1) >= k0 + kWaveKeys - 1)) {
      products(tile, 0, s0, [](int) {});
      products(tile, 1, s1, [&](int i) {
        add(s0, i * 32 / kSteps, (i + 1) * 32 / kSteps, c, l0);
      });
      add(s1, 0, 32, c, l1);
      return;
    }
#pragma unroll 1
    for (int ct = 0; ct < 2; ++ct) {
      const float lse = ct ? l1 : l0;
      const int pos = max(-1, ct ? p1 : p0), seen = pos - k0 - 4 * half;
      if (!__any(pos >= k0)) continue;
      products(tile, ct, s0, [](int) {});
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        const float x = __builtin_amdgcn_exp2f(fmaf(s0[e / 16][e % 16], c, -lse));
        sum[e] += 32 * (e / 16) + 8 * (e % 16 / 4) + e % 4 <= seen ? x : 0.0f;
      }
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
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1)
void kv_weigh_kernel(KvWeighArgs a, int chunks) {
  using W = Weigh<DP, BF16>;
  using Tile = typename W::Tile;
  __shared__ Tile tiles[kStages];
  const int h = (int)(blockIdx.x % a.c.heads);
  const int64_t rest = blockIdx.x / a.c.heads;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  int64_t piece = 0;
  int r = (int)(rest / chunks), base = -1;
  if (a.piece) {
    const Work work = work_of(a);
    const int p = r, requests = (int)a.q.requests;
    if (p >= work.first[requests]) return;
    r = uniform(below(requests, lane, [&](int i) { return work.first[i]; }, p + 1)) - 1;
    piece = p - uniform(work.first[r]);
    base = uniform(work.base[r]);
  }
  Span sp = span_of(a, r);
  sp = {uniform(sp.begin), uniform(sp.tokens), uniform(sp.first), uniform(sp.last)};
  const int32_t* table = a.q.table + r * a.q.table_stride;
  float* mass = a.mass + ((int64_t)r * a.c.heads + h) * a.slots;
  const float c = a.scale * kLog2e;
  W w(a, h);
  for (int64_t chunk = rest % chunks; chunk * kChunk <= sp.last; chunk += chunks) {
    // the tokens that see the chunk, of the piece's
    const int first = (int)(chunk * kChunk), k0 = first + wave * kWaveKeys;
    const int blind = uniform(
        below(sp.tokens, lane, [&](int i) { return a.q.positions[sp.begin + i]; }, first));
    const int x0 = base < 0 ? blind : (int)max((int64_t)blind, piece * a.piece);
    const int x1 = base < 0 ? sp.tokens : (int)min((int64_t)sp.tokens, (piece + 1) * a.piece);
#pragma unroll
    for (int e = 0; e < 32; ++e) w.sum[e] = 0.0f;
    if (x0 < x1) {
      w.start(sp.begin + x0, sp.begin + x1);
      const int todo = w.tiles();
#pragma unroll
      for (int n = 0; n < kStages - 1; ++n) w.copy(tiles[n]);
      w.keys(table, k0, sp.last);
      // (known to the compiler, which else waits for the keys, and with them for all
      // that was loaded since, in every turn)
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
#pragma unroll 1
      for (int n = 0; n < todo; ++n) {
        staged_barrier<(kStages - 2) * W::kLoads>();
        w.copy(tiles[(n + kStages - 1) % kStages]);  // (the place of the one before)
        if (k0 <= sp.last) w.use(tiles[n % kStages], k0, c);
      }
      dma_barrier();  // (nothing is on its way into the tiles any more)
      mfma_settle();
    }
    const float got = w.meet();
    const int p = k0 + W::key_of(lane);
    if (p > sp.last) continue;
    if (base >= 0) {
      const int64_t keys = (int64_t)a.q.cols << a.c.lps;
      work_of(a).sums[((base + piece) * a.c.heads + h) * keys + p] = got;
    } else {
      const int page = table[p >> a.c.lps];
      put(a, mass, p, sp.first, page >= 0 && page < a.c.pages ? got : 0.0f);
    }
  }
}

// Adds up the pieces of a request's sums, in their order.
__global__ __launch_bounds__(256) void kv_weigh_join_kernel(KvWeighArgs a, int blocks) {
  const Work work = work_of(a);
  const int h = (int)(blockIdx.x % a.c.heads);
  const int64_t rest = blockIdx.x / a.c.heads;
  if (rest / blocks >= work.count[0]) return;
  const int64_t r = work.several[rest / blocks];
  const Span sp = span_of(a, r);
  const int pieces = (int)pieces_of(a, sp.tokens);
  const int64_t keys = (int64_t)a.q.cols << a.c.lps;
  const float* sums = work.sums + ((int64_t)work.base[r] * a.c.heads + h) * keys;
  for (int64_t p = rest % blocks * 256 + threadIdx.x; p <= sp.last; p += (int64_t)blocks * 256) {
    float got = 0.0f;
#pragma unroll 4
    for (int i = 0; i < pieces; ++i) got += sums[i * a.c.heads * keys + p];
    const int page = a.q.table[r * a.q.table_stride + (p >> a.c.lps)];
    put(a, a.mass + (r * a.c.heads + h) * a.slots, (int)p, sp.first,
        page >= 0 && page < a.c.pages ? got : 0.0f);
  }
}

int64_t chunks_of(const KvWeighArgs& a) {
  const int64_t most = std::min<int64_t>(a.longest, (int64_t)a.q.cols << a.c.lps);
  return std::max<int64_t>(1, (most + kChunk - 1) / kChunk);
}

// At most so many pieces of all requests, partial sums, and requests that have some.
struct Most {
  int64_t pieces, sums, several;
};
Most most_of(const KvWeighArgs& a) {
  if (!a.piece) return {a.q.requests, 0, 0};
  const int64_t full = a.q.tokens / a.piece;
  return {a.q.requests + full, 2 * full, std::min(a.q.requests, full)};
}

template <int DP, bool BF16>
void launch_dim(const KvWeighArgs& a, hipStream_t s) {
  const int64_t chunks = chunks_of(a), grid = most_of(a).pieces * chunks * a.c.heads;
  kv_weigh_kernel<DP, BF16><<<dim3((unsigned)grid), 256, 0, s>>>(a, (int)chunks);
}

template <bool BF16>
void launch_type(const KvWeighArgs& a, hipStream_t s) {
  if (a.c.dim <= 64) launch_dim<64, BF16>(a, s);
  else if (a.c.dim <= 96) launch_dim<96, BF16>(a, s);
  else if (a.c.dim <= 128) launch_dim<128, BF16>(a, s);
  else if (a.c.dim <= 192) launch_dim<192, BF16>(a, s);
  else launch_dim<256, BF16>(a, s);
}

constexpr int64_t kUnits = 2048;
constexpr int64_t kLeast = 1024;  // rows of a piece

}  // namespace

void kv_weigh_plan(KvWeighArgs& a) {
  const int64_t pieces = std::max<int64_t>(1, kUnits / (chunks_of(a) * a.c.heads));
  const int64_t each = std::max<int64_t>(1, kRows / a.q.group);  // tokens of a tile
  const int64_t piece = std::max((a.q.tokens + pieces - 1) / pieces, kLeast / a.q.group);
  a.piece = (piece + each - 1) / each * each;
  if (a.piece >= a.q.tokens) a.piece = 0;
}

int64_t kv_weigh_workspace(const KvWeighArgs& a) {
  if (!a.piece) return 0;
  return 4 * (header_ints(a) + most_of(a).sums * a.c.heads * ((int64_t)a.q.cols << a.c.lps));
}

int64_t kv_weigh_grid(const KvWeighArgs& a) {
  return most_of(a).pieces * chunks_of(a) * a.c.heads;
}

hipError_t launch_kv_weigh(const KvWeighArgs& a, hipStream_t s) {
  if (a.piece) {
    kv_weigh_plan_kernel<<<1, kPlanThreads, 0, s>>>(a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  a.c.bf16 ? launch_type<true>(a, s) : launch_type<false>(a, s);
  if (hipError_t e = hipGetLastError(); e != hipSuccess || !a.piece) return e;
  const int64_t blocks = chunks_of(a), grid = most_of(a).several * blocks * a.c.heads;
  kv_weigh_join_kernel<<<dim3((unsigned)grid), 256, 0, s>>>(a, (int)blocks);
  return hipGetLastError();
}

}  // namespace mlxvs::kern
