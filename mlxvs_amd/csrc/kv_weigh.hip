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
// head each) come through LDS by direct loads, 64 at a time, one tile ahead, for
// all four wavefronts.  A lane adds up its column's weights of each of its 32 keys
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
  return max((int64_t)1, ((int64_t)tokens * a.q.group + a.piece - 1) / a.piece);
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

__device__ const uintx4 kZeros = {};  // what rows have past the head

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
  __device__ __forceinline__ static int swap(int row) {
    return kRow == 8 ? row >> 1 & 7 : row & 15;
  }

  struct Info {
    float lse;  // times log2(e); infinity for a row that is not there
    int pos;
  };

  const KvWeighArgs& a;
  const int lane, wave, h, group;
  // the row of the next tile that this thread (of the first wavefront) prepares
  uint32_t x, end;       // which row of the request's, of how many
  int token, head, begin;  // its token and head there; the request's first token
  // the chunk that this lane copies of its rows: they are 16 apart, or 8, whose
  // chunks' places differ
  static constexpr int kFrom = kRow == 32 ? 2 : 1;
  int from[kFrom];
  uintx4 kf[2][kSteps];
  float sum[32];

  __device__ __forceinline__ Weigh(const KvWeighArgs& args, int hd)
      : a(args), lane(threadIdx.x & 63), wave(threadIdx.x >> 6), h(hd), group(args.q.group) {
#pragma unroll
    for (int i = 0; i < kFrom; ++i) {
      const int slot = (wave + 4 * i) * 64 + lane, chunk = (slot % kRow) ^ swap(slot / kRow);
      from[i] = 8 * chunk < a.c.dim ? 8 * chunk : -1;
    }
  }

  // Rows x0 .. x1 - 1 of a request.
  __device__ __forceinline__ void start(int first_token, int64_t x0, int64_t x1) {
    begin = first_token;
    end = (uint32_t)x1;
    x = (uint32_t)x0 + lane;
    token = (int)(x / group);
    head = (int)(x % group);
  }

  // The first wavefront: where the next tile's rows begin (those past the last are
  // the last one).
  __device__ __forceinline__ void address(int64_t* to) {
    const uint32_t last = end - 1;
    const bool there = x < end;
    const int t = there ? token : (int)(last / group), g = there ? head : (int)(last % group);
    to[lane] = (int64_t)(begin + t) * a.q.q_token + (int64_t)(h * group + g) * a.q.q_head;
  }
  // ... and what the columns need of them, before it goes on by a tile.
  __device__ __forceinline__ Info info() {
    Info n{__builtin_inff(), -1};
    if (x < end) {
      const int64_t t = begin + token;
      n.lse = a.lse[t * a.c.heads * group + h * group + head];
      n.pos = max(-1, a.q.positions[t]);
    }
    x += kRows;
    token += kRows / group;
    head += kRows % group;
    if (head >= group) {
      head -= group;
      ++token;
    }
    return n;
  }

  // Copies a tile into LDS.
  __device__ __forceinline__ void copy(const int64_t* rows, char* to) const {
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int f = from[i % kFrom];
      const T* src = (const T*)a.q.q + rows[((wave + 4 * i) * 64 + lane) / kRow] + f;
      copy16_to_lds(f >= 0 ? (const void*)src : &kZeros, to + 1024 * (wave + 4 * i));
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
  __device__ __forceinline__ void products(const char* tile, int ct, floatx16 (&s)[2],
                                           Between between) const {
    const int col = lane & 31, half = lane >> 5;
    const char* at = tile + (32 * ct + col) * kRow * 16;
    const int sw = half ^ swap(32 * ct + col);
    uintx4 q[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) q[i] = *(const uintx4*)(at + 16 * (sw ^ (2 * i)));
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
  __device__ __forceinline__ void use(const char* tile, const Info* info, int k0, float c) {
    const int col = lane & 31, half = lane >> 5;
    const Info n0 = info[col], n1 = info[32 + col];
    floatx16 s0[2], s1[2];
    if (__all(min(n0.pos, n1.pos) >= k0 + kWaveKeys - 1)) {
      products(tile, 0, s0, [](int) {});
      products(tile, 1, s1, [&](int i) {
        add(s0, i * 32 / kSteps, (i + 1) * 32 / kSteps, c, n0.lse);
      });
      add(s1, 0, 32, c, n1.lse);
      return;
    }
#pragma unroll 1
    for (int ct = 0; ct < 2; ++ct) {
      const float lse = ct ? n1.lse : n0.lse;
      const int pos = ct ? n1.pos : n0.pos, seen = pos - k0 - 4 * half;
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
  using Info = typename W::Info;
  __shared__ __align__(16) char t0[W::kTileBytes], t1[W::kTileBytes];
  __shared__ Info i0[kRows], i1[kRows];
  __shared__ int64_t r0[kRows], r1[kRows];
  const int h = (int)(blockIdx.x % a.c.heads);
  const int64_t rest = blockIdx.x / a.c.heads;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t r = rest / chunks, base = -1;
  int piece = 0;
  if (a.piece) {
    const Work work = work_of(a);
    const int p = (int)r, requests = (int)a.q.requests;
    if (p >= work.first[requests]) return;
    r = below(requests, lane, [&](int i) { return work.first[i]; }, p + 1) - 1;
    piece = p - work.first[r];
    base = work.base[r];
  }
  const Span sp = span_of(a, r);
  const int32_t* table = a.q.table + r * a.q.table_stride;
  float* mass = a.mass + (r * a.c.heads + h) * a.slots;
  const int64_t rows = (int64_t)sp.tokens * a.q.group;
  const float c = a.scale * kLog2e;
  W w(a, h);
  for (int64_t chunk = rest % chunks; chunk * kChunk <= sp.last; chunk += chunks) {
    // the rows that see the chunk, of the piece's
    const int from = (int)(chunk * kChunk), k0 = from + wave * kWaveKeys;
    const int blind = below(sp.tokens, lane, [&](int i) { return a.q.positions[sp.begin + i]; }, from);
    const int64_t x0 = max((int64_t)blind * a.q.group, base < 0 ? 0 : piece * a.piece);
    const int64_t x1 = base < 0 ? rows : min(rows, (piece + 1) * a.piece);
    w.keys(table, k0, sp.last);
#pragma unroll
    for (int e = 0; e < 32; ++e) w.sum[e] = 0.0f;
    if (x0 < x1) {
      w.start(sp.begin, x0, x1);
      const bool tells = wave == 0;
      const auto tell = [&](Info* to, Info n) { to[lane] = {n.lse * kLog2e, n.pos}; };
      int todo = (int)((x1 - x0 + kRows - 1) / kRows);
      const auto turn = [&](char* tile, Info* info, int64_t* rows, char* other, Info* then,
                            int64_t* next) {
        dma_barrier();  // this tile is there, and the other buffer is free
        Info n{};
        const bool more = --todo > 0;
        if (more) {
          w.copy(next, other);
          if (tells) {
            n = w.info();
            w.address(rows);
          }
        }
        if (k0 <= sp.last) w.use(tile, info, k0, c);
        if (more && tells) tell(then, n);
      };
      __syncthreads();  // (the last chunk's buffers are free)
      if (tells) {
        w.address(r0);
        tell(i0, w.info());
        w.address(r1);
      }
      __syncthreads();
      w.copy(r0, t0);
      while (todo > 0) {
        turn(t0, i0, r0, t1, i1, r1);
        if (todo > 0) turn(t1, i1, r1, t0, i0, r0);
      }
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
  const int64_t full = a.q.tokens * a.q.group / a.piece;
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
  const int64_t rows = a.q.tokens * a.q.group, units = chunks_of(a) * a.c.heads;
  const int64_t pieces = std::max<int64_t>(1, kUnits / units);
  const int64_t piece = std::max(kLeast, ((rows + pieces - 1) / pieces + kRows - 1) / kRows * kRows);
  a.piece = piece < rows ? piece : 0;
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
