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
// its column's weights of each of its 32 keys over all rows, and the columns meet
// once at the end.  A product of 32 x 32 takes 33 cycles of a SIMD, the 6 vector
// instructions of its 2 weights a lane (fma, exp, add) 21, so both kinds are written
// side by side, a block's products next to the weights of the one before: 41 cycles,
// 59 if four of each follow one another.
//
// Measured: single tokens over 64 requests of up to 8,192 keys in 8 heads of 128
// values 122 us, 5.1 TB/s of keys, masses and their return (a copy: 4.95); chunks of
// 1,500 tokens in 3 requests of up to 8,192, 32 heads on 8, 138 us, 836 TFLOP/s, and
// a prompt of 4,001 tokens, 28 heads on 4, 86 us, 667 (16 prompts of up to 32,768
// together 875 to 891).  Two workgroups on a CU take 28 ns a product and SIMD, as a large
// library product does (27, the card's power); the rest are some 4 us at a unit's
// begin, until its keys and first rows are there, the end, where CUs run dry, masked
// tiles, and 12 us of plan and joining.  Tried: 128 keys a wavefront and 128 rows a
// tile, with one wavefront a SIMD, 181 and 144; one share of all tiles for each
// workgroup, which may go on in another chunk, 211 and 103 (the rows of Q then miss
// in L2); a fifth of the tiles in small units, the same.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "kv_cache.h"
#include "kv_mfma.h"
#include "lds_stage.h"

namespace mlxvs::kern {
namespace {

// x, which is the same in all lanes.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// A request's tokens of the step, and the keys that they see: token i of it those up
// to position first + i.
struct Span {
  int begin, tokens;
  int first, last;  // positions of the first and the last token; last -1: they see none
};

__device__ __forceinline__ Span span_of(const KvWeighArgs& a, int64_t r) {
  Span s;
  const int64_t lo = a.starts[r], hi = a.starts[r + 1];
  s.begin = (int)min(max(lo, (int64_t)0), a.q.tokens);
  s.tokens = (int)(min(max(hi, (int64_t)s.begin), a.q.tokens) - s.begin);
  s.first = s.last = -1;
  if (s.tokens > 0) {
    s.first = a.q.positions[s.begin];
    // (one that was not admitted has none; the table ends somewhere)
    const int64_t end = ((int64_t)a.q.cols << a.c.lps) - 1;
    if (s.first >= 0) s.last = (int)min((int64_t)s.first + s.tokens - 1, end);
  }
  return s;
}

// What a key got before, and gets now.
__device__ __forceinline__ void put(const KvWeighArgs& a, float* mass, int p, int first, float got) {
  const float before = p < first && a.decay != 0.0f ? a.decay * mass[p] : 0.0f;
  mass[p] = before + got;
}

// ---- single tokens -------------------------------------------------------------

constexpr int kFewKeys = 32;  // of a wavefront at a time, in two tiles of 16
// Keys of a workgroup of single tokens, 32 at a time for each of its wavefronts: 64
// requests of up to 8,192 keys with 128: 134 us, 256: 122, 512: 122, 1,024: 124.
constexpr int kSpan = 256;

// The sum over the 16 lanes of a row.
__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
  for (int i = 8; i >= 1; i >>= 1) x += __shfl_xor(x, i);
  return x;
}

// Requests of up to few_rows rows.  kSpan keys of a request and head a workgroup, 32 a
// wavefront at a time, the next ones on their way; with more keys than the `spans`
// workgroups of a request and head hold it comes again.
// The rows of up to 16 query heads stay in registers.
template <int DP, bool BF16>
__global__ __launch_bounds__(256) void kv_weigh_few_kernel(KvWeighArgs a, int spans) {
  using T = std::conditional_t<BF16, __bf16, _Float16>;
  using Tx8 = std::conditional_t<BF16, bf16x8, halfx8>;
  constexpr int kSteps = DP / 32;
  struct Keys {
    uintx4 k[2][kSteps];
    bool there[2];
    float mass;  // of the lane's key, before
  };
  struct Rows {
    uintx4 q[kSteps];
    float lse;
    int pos;
  };
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), col = lane & 15, grp = lane >> 4;
  const int d = a.c.dim, group = a.q.group;
  const int h = (int)(blockIdx.x % a.c.heads);
  const int64_t rest = blockIdx.x / a.c.heads;
  const int r = (int)(rest % a.q.requests);
  Span sp = span_of(a, r);
  sp = {uniform(sp.begin), uniform(sp.tokens), uniform(sp.first), uniform(sp.last)};
  const int32_t* table = a.q.table + (int64_t)r * a.q.table_stride;
  float* mass = a.mass + ((int64_t)r * a.c.heads + h) * a.slots;
  const int64_t rows = (int64_t)sp.tokens * group;
  if (rows > a.few_rows) return;

  const auto load_rows = [&](int64_t x0, Rows& y) {
    const int64_t x = x0 + col;
    const bool mine = x < rows;
    const int64_t t = sp.begin + (mine ? x / group : 0);
    const int g = h * group + (mine ? (int)(x % group) : 0);
    y.pos = mine ? (int)min(sp.first + x / group, (int64_t)sp.last) : -1;
    y.lse = a.lse[t * a.c.heads * group + g];
    const T* src = (const T*)a.q.q + t * a.q.q_token + g * a.q.q_head + 8 * grp;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      y.q[i] = uintx4{};
      if (32 * i + 32 <= sure_values(DP) || 32 * i + 8 * grp < d) y.q[i] = *(const uintx4*)(src + 32 * i);
    }
  };
  const auto key_of = [&](int k0) { return k0 + 16 * (lane >> 5) + 4 * (lane >> 3 & 3) + (lane & 3); };
  const auto pages = [&](int64_t k0, int (&page)[2]) {
#pragma unroll
    for (int u = 0; u < 2; ++u) page[u] = k0 + 16 * u <= sp.last ? table[(k0 + 16 * u) >> a.c.lps] : -1;
  };
  const auto load = [&](int k0, const int (&page)[2], Keys& y) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      y.there[u] = page[u] >= 0 && page[u] < a.c.pages;
      const T* row = (const T*)a.c.keys +
                     (((int64_t)(y.there[u] ? page[u] : 0) * a.c.heads + h) * a.c.page +
                      ((k0 + 16 * u) & (a.c.page - 1)) + col) * d + 8 * grp;
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        y.k[u][i] = uintx4{};
        if (y.there[u] && (32 * i + 32 <= sure_values(DP) || 32 * i + 8 * grp < d))
          y.k[u][i] = *(const uintx4*)(row + 32 * i);
      }
    }
    const int p = key_of(k0);
    y.mass = 0.0f;
    if (!(lane & 4) && p < sp.first && p <= sp.last && a.decay != 0.0f) y.mass = mass[p];
  };
  const auto weigh = [&](const Keys& y, const Rows& z, int k0, float (&sum)[2][4]) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      floatx4 s = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < kSteps; ++i)
        s = mfma(__builtin_bit_cast(Tx8, y.k[u][i]), __builtin_bit_cast(Tx8, z.q[i]), s);
      const int seen = z.pos - (k0 + 16 * u + 4 * grp);  // keys up to this one
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = __builtin_amdgcn_exp2f(fmaf(s[i], a.scale, -z.lse) * kLog2e);
        sum[u][i] += i <= seen ? x : 0.0f;
      }
    }
  };

  const int64_t stride = (int64_t)spans * kSpan;
  for (int64_t at = rest / a.q.requests * kSpan; at <= sp.last; at += stride) {
    const int64_t end = min(at + kSpan, (int64_t)sp.last + 1);
    int64_t k0 = at + wave * kFewKeys;
    if (k0 >= end) return;
    int page[2];
    Keys one, two;
    pages(k0, page);
    Rows first;
    load_rows(0, first);
    load((int)k0, page, one);
    pages(k0 + 4 * kFewKeys, page);
    const auto turn = [&](Keys& now, Keys& then) {
      const int64_t next = k0 + 4 * kFewKeys;
      if (next < end) {
        load((int)next, page, then);
        pages(next + 4 * kFewKeys, page);
      }
      float sum[2][4] = {};
      weigh(now, first, (int)k0, sum);
      for (int64_t x0 = 16; x0 < rows; x0 += 16) {
        Rows more;
        load_rows(x0, more);
        if (__any(more.pos >= k0)) weigh(now, more, (int)k0, sum);
      }
      // lane l writes key_of: its tile's, its row's and one of the four
      float got[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        got[u] = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float all = row_sum(sum[u][i]);
          if ((lane & 3) == i) got[u] = now.there[u] ? all : 0.0f;
        }
      }
      const int p = key_of((int)k0), from = 16 * (lane >> 3 & 3) + (lane & 3);
      const float a0 = __shfl(got[0], from), a1 = __shfl(got[1], from);
      if (!(lane & 4) && p <= sp.last) mass[p] = a.decay * now.mass + (lane & 32 ? a1 : a0);
      k0 = next;
    };
    while (k0 < end) {
      turn(one, two);
      if (k0 < end) turn(two, one);
    }
  }
}

// ---- prompts -------------------------------------------------------------------

constexpr int kStages = 4;  // tiles in LDS: one in use, the others on their way

constexpr int kWaveKeys = 64, kChunk = 4 * kWaveKeys;  // keys of a wavefront, a workgroup
constexpr int kRows = 64;                              // of a tile of Q

// A workgroup's share: a chunk of a request's keys, and some tokens that see it.
struct Unit {
  int request, chunk;
  int begin, end;   // tokens of the batch
  int slot;         // where its sums go, -1: into the masses
  int shift, last;  // a token's position less its place in the batch; the last position
  int pieces;       // of the chunk, at its first unit: sums in as many slots
};

// The workspace, made by one workgroup: the units, and the first ones of chunks that
// several units share.
struct Work {
  int32_t* units;   // [1] how many there are, and chunks of several
  int32_t* shared;  // [1]
  int32_t* first;   // [requests + 1] chunks before a request's
  Unit* unit;
  Unit* several;
  float* sums;      // [slots][heads][kChunk]
};

__host__ __device__ __forceinline__ int64_t header_ints(const KvWeighArgs& a) {
  return (2 + a.q.requests + 1 + 3) / 4 * 4;
}
__device__ __forceinline__ Work work_of(const KvWeighArgs& a) {
  int32_t* w = a.work;
  Unit* unit = (Unit*)(w + header_ints(a));
  return {w, w + 1, w + 2, unit, unit + a.most_units, (float*)(unit + a.most_units + a.most_several)};
}

// A request's first position.
__device__ __forceinline__ int first_of(const KvWeighArgs& a, int r) { return span_of(a, r).first; }

constexpr int kPlanThreads = 1024;

// The sum over a workgroup's threads up to each one; `all` gets the total.
__device__ __forceinline__ int running(int x, int& all, int* waves) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int by = 1; by < 64; by <<= 1) {
    const int y = __shfl_up(x, by);
    if (lane >= by) x += y;
  }
  if (lane == 63) waves[wave] = x;
  __syncthreads();
  all = 0;
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    if (w < wave) x += waves[w];
    all += waves[w];
  }
  __syncthreads();
  return x;
}
// The first of a request's tokens that sees key p (its number of tokens: none).
__device__ __forceinline__ int sees(int first, int tokens, int64_t p) {
  return (int)min(max(p - first, (int64_t)0), (int64_t)tokens);
}

// Units over all heads, besides one for each chunk: two rounds of two workgroups a CU.
// The costly ones come first, as workgroups are not equally fast (of two on a CU the
// older one takes 1.5 us a tile, the other 2.15).  Chunks of 1,500 tokens and a prompt
// of 4,001 with 512: 155 and 99 us, 768: 141 and 93, 1,024: 138 and 86, 1,536: 145 and
// 93; with 1,024 in the chunks' order 150 and 94.
constexpr int kShares = 1024;
constexpr int kLeastTiles = 4;  // of a unit
constexpr int kClasses = 64;    // of units, by cost
__host__ __device__ __forceinline__ int more_units(const KvWeighArgs& a) {
  return kShares > a.c.heads ? kShares / a.c.heads : 1;
}

constexpr int kPlanSpans = 1024;  // requests whose spans stay in LDS

__global__ __launch_bounds__(kPlanThreads) void kv_weigh_plan_kernel(KvWeighArgs a) {
  constexpr int kWaves = kPlanThreads / 64;
  __shared__ int waves[kWaves];
  __shared__ Span spans[kPlanSpans];
  __shared__ int firsts[kPlanSpans + 1];
  __shared__ int64_t totals[kWaves];
  __shared__ int at[kClasses], several, slots;
  struct Cut {  // a chunk; masked: tiles of which a row does not see all keys
    int request, chunk, from, tiles, masked, units, slot;
  };
  __shared__ Cut cuts[kPlanThreads];
  __shared__ int ends[kPlanThreads];  // units up to a chunk's last
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Work work = work_of(a);
  const bool few = a.q.requests <= kPlanSpans;
  struct Part {  // a request's chunk, the first of its tokens that sees it
    int request, chunk;
    Span sp;
    int from;
  };
  const auto part = [&](int i) {
    int lo = 0, hi = (int)a.q.requests;  // first[lo] <= i < first[hi]
    while (hi - lo > 1) {
      const int mid = lo + (hi - lo) / 2;
      if ((few ? firsts[mid] : work.first[mid]) <= i) lo = mid;
      else hi = mid;
    }
    Part p{lo, i - (few ? firsts[lo] : work.first[lo]), few ? spans[lo] : span_of(a, lo), 0};
    p.from = min(sees(p.sp.first, p.sp.tokens, (int64_t)p.chunk * kChunk), p.sp.tokens - 1);
    return p;
  };
  const auto tiles_of = [&](const Part& p) { return (p.sp.tokens - p.from + a.tile - 1) / a.tile; };
  // the requests' chunks ...
  int chunks = 0;
  for (int64_t r0 = 0; r0 < a.q.requests; r0 += kPlanThreads) {
    const int64_t r = r0 + threadIdx.x;
    int n = 0, all;
    if (r < a.q.requests) {
      const Span sp = span_of(a, r);
      if (few) spans[r] = sp;
      const bool mine = sp.last >= 0 && (int64_t)sp.tokens * a.q.group > a.few_rows;
      n = mine ? sp.last / kChunk + 1 : 0;
    }
    n = running(n, all, waves);
    if (r < a.q.requests) {
      if (few) firsts[r + 1] = chunks + n;
      else work.first[r + 1] = chunks + n;
    }
    chunks += all;
  }
  if (threadIdx.x == 0) firsts[0] = work.first[0] = several = slots = 0;
  if (threadIdx.x < kClasses) at[threadIdx.x] = 0;
  __syncthreads();
  // ... how many tiles they have altogether ...
  int64_t total = 0;
  for (int i = threadIdx.x; i < chunks; i += kPlanThreads) total += tiles_of(part(i));
#pragma unroll
  for (int i = 32; i >= 1; i >>= 1) total += __shfl_xor(total, i);
  if (lane == 0) totals[wave] = total;
  __syncthreads();
  total = 0;
  for (int w = 0; w < kWaves; ++w) total += totals[w];
  const int extra = more_units(a);
  const int piece = (int)max((int64_t)kLeastTiles, (total + extra - 1) / extra);
  // ... and their units, of as many tiles or one less, the costly ones first
  const auto fill = [&](int i0, bool placing) {  // kPlanThreads chunks; their number of units
    const int i = i0 + threadIdx.x;
    Cut c{};
    if (i < chunks) {
      const Part p = part(i);
      const int tiles = tiles_of(p);
      const int all = sees(p.sp.first, p.sp.tokens, (int64_t)(p.chunk + 1) * kChunk - 1) - p.from;
      c = {p.request, p.chunk, p.from, tiles, min(tiles, (max(all, 0) + a.tile - 1) / a.tile),
           (tiles + piece - 1) / piece, -1};
      if (placing && c.units > 1) c.slot = atomicAdd(&slots, c.units);
    }
    int all;
    ends[threadIdx.x] = running(c.units, all, waves);
    cuts[threadIdx.x] = c;
    __syncthreads();
    return all;
  };
  const auto each = [&](int units, auto use) {  // (chunk, its how many-th unit)
    for (int u = threadIdx.x; u < units; u += kPlanThreads) {
      int lo = 0, hi = kPlanThreads - 1;  // the first one whose end is past u
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (ends[mid] > u) hi = mid;
        else lo = mid + 1;
      }
      const Cut c = cuts[lo];
      use(c, u - (ends[lo] - c.units));
    }
  };
  const auto edge = [&](const Cut& c, int j) {  // where unit j begins
    return c.tiles / c.units * j + min(j, c.tiles % c.units);
  };
  const auto class_of = [&](const Cut& c, int from, int to) {
    const float cost = (float)(to - from) + 0.3f * (float)min(max(c.masked - from, 0), to - from);
    return (int)((float)(kClasses - 1) * max(0.0f, 1.0f - cost / (1.3f * (float)piece)));
  };
  int units = 0;
  for (int i0 = 0; i0 < chunks; i0 += kPlanThreads) {
    if (i0 > 0) __syncthreads();  // (the last ones are done with)
    units = fill(i0, chunks <= kPlanThreads);
    each(units, [&](const Cut& c, int j) { atomicAdd(&at[class_of(c, edge(c, j), edge(c, j + 1))], 1); });
  }
  __syncthreads();
  if (wave == 0) {
    int n = lane < kClasses ? at[lane] : 0;
    const int own = n;
#pragma unroll
    for (int by = 1; by < 64; by <<= 1) {
      const int y = __shfl_up(n, by);
      if (lane >= by) n += y;
    }
    if (lane < kClasses) at[lane] = n - own;
    if (lane == 63) work.units[0] = n;
  }
  __syncthreads();
  // (which of a class comes first only changes where its sums are)
  for (int i0 = 0; i0 < chunks; i0 += kPlanThreads) {
    if (i0 > 0) __syncthreads();
    if (chunks > kPlanThreads) units = fill(i0, true);
    each(units, [&](const Cut& c, int j) {
      const Span sp = few ? spans[c.request] : span_of(a, c.request);
      const int from = edge(c, j), to = edge(c, j + 1);
      const Unit u{c.request, c.chunk, sp.begin + c.from + from * a.tile,
                   sp.begin + min(sp.tokens, c.from + to * a.tile), c.units > 1 ? c.slot + j : -1,
                   sp.first - sp.begin, sp.last, c.units};
      work.unit[atomicAdd(&at[class_of(c, from, to)], 1)] = u;
      if (j == 0 && c.units > 1) work.several[atomicAdd(&several, 1)] = u;
    });
  }
  __syncthreads();
  if (threadIdx.x == 0) work.shared[0] = several;
}

// What rows of a tile have past the head, and rows that are not the unit's: zeros, with
// a logarithm that leaves no weight.
__device__ const uintx4 kZeros = {};
__device__ const float kNoLse = __builtin_inff();

// DP: head size rounded up.
template <int DP, bool BF16>
struct Weigh {
  using T = std::conditional_t<BF16, __bf16, _Float16>;
  static constexpr int kSteps = DP / 16;
  // A tile in LDS: rows of 16-byte chunks, their logarithms, and 256 bytes that are not
  // read.  A chunk's place in its row is swapped so that 16 rows' same chunk lies in all
  // banks; tiles are aligned so that it is some bits of its address.
  static constexpr int kRow = DP <= 64 ? 8 : DP <= 128 ? 16 : 32;
  static constexpr int kLse = kRows * kRow * 16, kNone = kLse + 4 * kRows;
  static constexpr int kTileBytes = (kNone + 256 + 511) / 512 * 512;
  static constexpr int kCopies = kRow / 4;    // of 1 KB a wavefront and tile
  static constexpr int kLoads = kCopies + 1;  // ... and one of 256 bytes
  __device__ __forceinline__ static int swap(int row) {
    return kRow == 8 ? row >> 1 & 7 : row & 15;
  }

  const KvWeighArgs& a;
  const int lane, wave, h, group, tokens_tile;  // (a tile: all of some tokens' heads)
  int64_t rows[kCopies];       // this lane's pieces of a tile, in bytes from its first row on
  uint64_t tokens;             // which of the tile's tokens they are of, a byte each
  static constexpr int kNoToken = 255;  // none: zeros
  int told, told_token;        // the row whose logarithm it brings
  int of[2];                   // the tokens of this lane's columns
  int token, end;              // the next tile's first token, one past the last of all
  uintx4 kf[2][kSteps];
  float sum[32];

  __device__ __forceinline__ Weigh(const KvWeighArgs& args, int head)
      : a(args), lane(threadIdx.x & 63), wave(uniform(threadIdx.x >> 6)), h(head),
        group(args.q.group), tokens_tile(args.tile) {
    tokens = 0;
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int slot = (wave + 4 * i) * 64 + lane, j = slot / kRow, chunk = (slot % kRow) ^ swap(j);
      rows[i] = 2 * (j / group * a.q.q_token + j % group * a.q.q_head + 8 * chunk);
      const bool none = 8 * chunk >= a.c.dim || j / group >= tokens_tile;
      tokens |= (uint64_t)(none ? kNoToken : j / group) << 8 * i;
    }
    told_token = lane / group < tokens_tile ? lane / group : kNoToken;
    told = lane / group * a.c.heads * group + lane % group;
    of[0] = (lane & 31) / group;
    of[1] = (32 + (lane & 31)) / group;
  }

  // Tokens t0 .. t1 - 1 of the batch; returns their tiles.
  __device__ __forceinline__ int start(int t0, int t1) {
    token = t0;
    end = t1;
    return (t1 - t0 + tokens_tile - 1) / tokens_tile;
  }

  // The next tile's copy into LDS (past the last: zeros), kLoads loads, one by one.
  struct Copy {
    const char* q;
    int left;  // tokens
    uint32_t to;
  };
  __device__ __forceinline__ Copy next(uint32_t tile) const {
    return {(const char*)a.q.q + 2 * (token * a.q.q_token + (int64_t)h * group * a.q.q_head),
            end - token, tile};
  }
  __device__ __forceinline__ void copy(const Copy& n, int i) {
    if (i < kCopies) {
      const bool there = (int)(tokens >> 8 * i & 255) < min(n.left, kNoToken);
      stream16_to_lds(there ? (const void*)(n.q + rows[i]) : &kZeros, n.to + 1024 * (wave + 4 * i));
      return;
    }
    // one wavefront brings the rows' logarithms, the others as much of nothing, so that
    // all have as many loads on their way
    const float* lse = a.lse + ((int64_t)token * a.c.heads + h) * group + told;
    stream4_to_lds(told_token < min(n.left, kNoToken) ? lse : &kNoLse,
                   n.to + (wave == 0 ? kLse : kNone));
    token = min(token + tokens_tile, end);
  }
  __device__ __forceinline__ void copy_all(uint32_t tile) {
    const Copy n = next(tile);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) copy(n, i);
  }

  // The keys from k0 on of a table's row.  (Where there is none some key of the cache
  // is read, whose sum is left out: a cache without pages does not come here.)
  __device__ __forceinline__ void keys(const int32_t* table, int k0, int upto) {
    const int d = a.c.dim, col = lane & 31, half = lane >> 5;
    int page[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) page[u] = table[min(k0 + 32 * u + col, upto) >> a.c.lps];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int k = k0 + 32 * u + col;
      const int64_t p = page[u] >= 0 && page[u] < a.c.pages ? page[u] : 0;
      const T* src = (const T*)a.c.keys + ((p * a.c.heads + h) * a.c.page + (k & (a.c.page - 1))) * d;
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const int at = 16 * i + 8 * half;
        if (16 * i + 16 <= sure_values(DP)) {
          kf[u][i] = *(const uintx4*)(src + at);
        } else {
          kf[u][i] = uintx4{};
          if (at < d) kf[u][i] = *(const uintx4*)(src + at);
        }
      }
    }
  }

  // Once they are there: keys of more than 128 values stay in accumulation registers,
  // which products read and vector instructions do not.  (With two wavefronts on a
  // SIMD it is better not to use any: the compiler then has all 256 registers for the
  // rest, and with some only half of them.)
  static constexpr bool kHeld = DP > 128;
  __device__ __forceinline__ void hold() {
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        if constexpr (kHeld) asm volatile("" : "+a"(kf[u][i]));
        else asm volatile("" : "+v"(kf[u][i]));
      }
#endif
  }

  // Where the lane's column (row 32 ct + lane % 32 of the tile) begins.
  __device__ __forceinline__ uint32_t column(uint32_t tile, int ct) const {
    const int row = 32 * ct + (lane & 31);
    return tile + row * kRow * 16 + 16 * ((lane >> 5) ^ swap(row));
  }

  // s (+)= keys x rows.  (Written out: left to itself the compiler has the sums in
  // accumulation registers, from where every value is moved before it is used.)
  template <bool FIRST>
  __device__ __forceinline__ static void product(floatx16& s, const uintx4& k, const uintx4& q) {
#if defined(__HIP_DEVICE_COMPILE__)
#define MLXVS_PRODUCT(TYPE, K)                                                              \
  if constexpr (FIRST)                                                                      \
    asm volatile("v_mfma_f32_32x32x16_" TYPE " %0, %1, %2, 0" : "=&v"(s) : K(k), "v"(q));   \
  else asm volatile("v_mfma_f32_32x32x16_" TYPE " %0, %1, %2, %0" : "+v"(s) : K(k), "v"(q))
    if constexpr (kHeld && BF16) { MLXVS_PRODUCT("bf16", "a"); }
    else if constexpr (kHeld) { MLXVS_PRODUCT("f16", "a"); }
    else if constexpr (BF16) { MLXVS_PRODUCT("bf16", "v"); }
    else { MLXVS_PRODUCT("f16", "v"); }
#undef MLXVS_PRODUCT
#endif
  }
  // Wait states before the sums are read, which the compiler does not count (12 of
  // them after a product of 8 passes).
  __device__ __forceinline__ static void settle() {
#if defined(__HIP_DEVICE_COMPILE__)
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 15");
    __builtin_amdgcn_sched_barrier(0);
#endif
  }

  // A block of products, 32 rows by 64 keys, whose weights are to be taken.
  struct Block {
    floatx16 s[2];
    float lse;  // times log2(e)
    int seen;   // the last of the keys that the lane's column sees, less 4 (lane / 32)
  };

  // The weights of a block, some for each of the next one's products; each is added a
  // step after it is made.  (The sums are tied to their place: they would be moved
  // behind all products, which then have nothing beside them.)
  static constexpr int kPer = (32 + 2 * kSteps - 1) / (2 * kSteps);
  static constexpr int kTurns = (32 + kPer - 1) / kPer;  // ... and one to add the last
  template <bool MASK>
  __device__ __forceinline__ void weigh(const Block& b, int i, float c, float (&x)[kPer]) {
    if (i > 0) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int e = (i - 1) * kPer + j;
        if (e >= 32) continue;
        sum[e] += x[j];
#if defined(__HIP_DEVICE_COMPILE__)
        asm volatile("" : "+v"(sum[e]));
#endif
      }
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int e = i * kPer + j;
      if (e >= 32) continue;
      x[j] = __builtin_amdgcn_exp2f(fmaf(b.s[e / 16][e % 16], c, -b.lse));
      if (MASK) x[j] = 32 * (e / 16) + 8 * (e % 16 / 4) + e % 4 <= b.seen ? x[j] : 0.0f;
    }
  }

  // The products of 32 rows with the keys, and beside them the weights of the block
  // before: one product and 6 vector instructions take as long.  Block B of a tile; its
  // rows' next values are read while the last ones are used, and also(i) does something
  // else beside the i-th product.
  static constexpr int kAhead = 4;
  template <int B, bool MASK, typename Also>
  __device__ __forceinline__ void products(uint32_t t, uintx4 (&q)[kAhead], Block& now,
                                           const Block& before, float c, Also also) {
    float x[kPer];
#pragma unroll
    for (int i = 0; i < 2 * kSteps; ++i) {
      constexpr int at = B * kSteps;
      uintx4& rows = q[(at + i / 2) % kAhead];
      if (i < 2) product<true>(now.s[i], kf[i][0], rows);
      else product<false>(now.s[i % 2], kf[i % 2][i / 2], rows);
      __builtin_amdgcn_sched_barrier(0);
      if (i <= kTurns) weigh<MASK>(before, i, c, x);
      if (const int n = at + i / 2 + kAhead; i % 2 && n < 2 * kSteps)
        rows = lds_read16(column(t, n / kSteps) ^ (32 * (n % kSteps)));
      also(i);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (2 * kSteps <= kTurns) weigh<MASK>(before, kTurns, c, x);
    // (the next block's first weights read sums whose last product has another one and
    // two products' vector instructions behind it: wait states enough, if there are some)
    if constexpr (6 * kPer + 2 < 14 || kTurns < 2 * kSteps) settle();
  }

  // Tiles from `from` to `to`, of which token t is `seen` + t - token.  Without MASK every
  // row sees every key (or is none).
  template <bool MASK, typename Tile, typename Wait>
  __device__ __forceinline__ void use(int from, int to, int k0, int shift, float c, Tile tile,
                                      Wait wait) {
    if (from >= to) return;
    constexpr int kEach = (kLoads + 1) / 2;  // copies beside a block
    constexpr int kApart = 2 * kSteps / kEach;
    Block open;
    open.s[0] = open.s[1] = floatx16{};
    open.lse = __builtin_inff();
    open.seen = 0;
#pragma unroll 1
    for (int n = from; n < to; ++n) {
      wait();
      const Copy then = next(tile(n + kStages - 1));  // (the place of the one before)
      const uint32_t t = tile(n);
      uintx4 q[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) q[i] = lds_read16(column(t, 0) ^ (32 * i));
      const float l0 = lds_read4<float>(t + kLse + 4 * (lane & 31)),
                  l1 = lds_read4<float>(t + kLse + 128 + 4 * (lane & 31));
      // (the tile's first token's position, less the keys that are not this lane's)
      const int pos = shift + n * tokens_tile - k0 - 4 * (lane >> 5);
      const auto also = [&](int block, int i) {
        if (i % kApart == kApart - 1 && i / kApart < kEach && block * kEach + i / kApart < kLoads)
          copy(then, block * kEach + i / kApart);
      };
      Block now;
      now.lse = l0 * kLog2e;
      now.seen = pos + of[0];
      products<0, MASK>(t, q, now, open, c, [&](int i) { also(0, i); });
      products<1, MASK>(t, q, open, now, c, [&](int i) { also(1, i); });
      open.lse = l1 * kLog2e;
      open.seen = pos + of[1];
    }
    settle();
    float x[kPer];
#pragma unroll
    for (int i = 0; i <= kTurns; ++i) weigh<MASK>(open, i, c, x);
  }

  // The sums over the columns: lane l's key is key_of(l).
  template <int B>
  __device__ __forceinline__ void halve(float (&x)[32]) const {
    const bool up = lane & B;
#pragma unroll
    for (int j = 0; j < B; ++j) {
      const float mine = up ? x[j + B] : x[j], other = up ? x[j] : x[j + B];
      x[j] = mine + __shfl_xor(other, B);
    }
  }
  __device__ __forceinline__ float meet() const {
    float x[32];
#pragma unroll
    for (int e = 0; e < 32; ++e) x[e] = sum[e];
    halve<16>(x);
    halve<8>(x);
    halve<4>(x);
    halve<2>(x);
    halve<1>(x);
    return x[0];
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
  const float c = __builtin_bit_cast(float, uniform(__builtin_bit_cast(int, a.scale * kLog2e)));
  const auto tile = [&](int n) { return at + n % kStages * W::kTileBytes; };
  const auto wait = [] {
    staged_barrier<(kStages - 2) * W::kLoads>();
    mfma_settle();
  };
  W w(a, h);
  for (int x = (int)(blockIdx.x / a.c.heads); x < units; x += (int)(gridDim.x / a.c.heads)) {
    const Unit u = work.unit[x];
    const int r = uniform(u.request), last = uniform(u.last), slot = uniform(u.slot);
    const int begin = uniform(u.begin), end = uniform(u.end), shift = uniform(u.shift);
    const int k0 = uniform(u.chunk) * kChunk + w.wave * kWaveKeys;
    const int32_t* table = a.q.table + r * a.q.table_stride;
#pragma unroll
    for (int e = 0; e < 32; ++e) w.sum[e] = 0.0f;
    const int todo = w.start(begin, end);
    w.keys(table, k0, last);
#pragma unroll
    for (int n = 0; n < kStages - 1; ++n) w.copy_all(tile(n));
    // (known to the compiler, which else waits for the keys, and with them for all
    // that was loaded since, in every turn)
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    w.hold();
    // the tiles of which some rows see some of this wavefront's keys, and those of which
    // all rows see all
    const int position = shift + begin;  // of the first token
    const int some = k0 > last ? todo : min(todo, sees(position, end - begin, k0) / w.tokens_tile);
    const int all = max(some, min(todo, (sees(position, end - begin, (int64_t)k0 + kWaveKeys - 1) +
                                         w.tokens_tile - 1) / w.tokens_tile));
#pragma unroll 1
    for (int n = 0; n < some; ++n) {
      wait();
      w.copy_all(tile(n + kStages - 1));
    }
    w.template use<true>(some, all, k0, position, c, tile, wait);
    w.template use<false>(all, todo, k0, position, c, tile, wait);
    dma_barrier();  // (nothing is on its way into the tiles any more)
    mfma_settle();
    const float got = w.meet();
    const int key = W::key_of(lane), p = k0 + key;
    if (p > last) continue;
    if (slot >= 0) {
      work.sums[((int64_t)slot * a.c.heads + h) * kChunk + w.wave * kWaveKeys + key] = got;
    } else {
      const int page = table[p >> a.c.lps];
      put(a, a.mass + ((int64_t)r * a.c.heads + h) * a.slots, p, first_of(a, r),
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
    put(a, a.mass + ((int64_t)u.request * a.c.heads + h) * a.slots, p, first_of(a, u.request),
        page >= 0 && page < a.c.pages ? got : 0.0f);
  }
}

// ---- which one ------------------------------------------------------------------

// Chunks of so many keys that requests are expected to have.
int64_t chunks_of(const KvWeighArgs& a, int64_t chunk, int64_t most) {
  most = std::min<int64_t>(most, (int64_t)a.q.cols << a.c.lps);
  return std::max<int64_t>(1, (most + chunk - 1) / chunk);
}

// Where there are more tokens than requests, at least 16 requests are dealt by their
// rows, those of up to 32 to the kernel of single tokens (a launch more).  All by the
// kernel of prompts / dealt: 64 requests of up to 8,192 keys, group 4, with 2 tokens each
// 217 / 151 us, with 8 214 / 193, with 12 215 / 227, 63 single tokens and a prompt of 512
// 233 / 185; 3 and that 48 / 55.
constexpr int kSomeRequests = 16, kFewRows = 32;

constexpr int64_t kGrid = 2048;  // workgroups at most

// Keys that a call's tables have room for, or that its requests are told to hold, in all
// heads.
int64_t room_of(const KvWeighArgs& a) {
  const int64_t rows = std::min<int64_t>(a.q.requests * a.c.heads, 1 << 30);
  return rows * std::min<int64_t>(a.longest, (int64_t)a.q.cols << a.c.lps);
}

// No more tokens than rows of the table are a token each, or a prompt among idle rows,
// which the device finds: where single tokens could take 0.4 ms or more, requests are
// dealt here, too.  By the kernel of single tokens / dealt (8 kv heads of 4, 128 values):
// a prompt of 200 tokens over 4,096 keys in a table of 512 rows 179 / 41 us (29 in one of
// its own), with a token in each other one, 1,000 keys, 377 / 233; 512 tokens over 16,384
// 1,134 / 105 (93).  No prompt, 256 rows of 4,096 keys 397 / 408, 1,024 1,612 / 1,622.
// More requests than these take the plan too long, 2 us for each turn: 131,072 of 64 keys
// 4,287 / 4,527, 16,384 538 / 576, 2,048 of 512 398 / 415.
constexpr int64_t kDealt = 8 << 20, kDealtRequests = kPlanSpans;

bool idle_rows(const KvWeighArgs& a) { return a.q.tokens <= a.q.requests; }

// Rows of queries that are few; of idle rows' tables a single token's, whatever they are
// (256 of 33 and 64 query heads over 32,768 keys of one kv head 565 and 685 us, by the
// kernel of prompts 899 and 902).
int64_t few_rows_of(const KvWeighArgs& a) {
  return idle_rows(a) ? std::max(kFewRows, a.q.group) : kFewRows;
}

// Whether a request may have more.
bool some_many(const KvWeighArgs& a) { return a.q.tokens * a.q.group > few_rows_of(a); }

// Workgroups of single tokens for each request and head: no more than make kFewGrid, as a
// table may be far wider than its requests are long; the rest of the keys is come to
// later.  Without a limit / with it, longest not told: 256 requests of up to 2,048 tokens
// in a table for 131,072 838 / 158 us (in one for 2,048 137), 1,024 of 1,000 in one for
// 32,768 1,117 / 432, 8 of up to 8,192 in one for 1,048,576 193 / 27.  (32,768: 165, 450,
// 38, and 1,024 of 4,096 1,649 instead of 1,623.)
constexpr int64_t kFewGrid = 16384;
// Many where there may be a prompt that is not dealt, which would have to do with a few:
// 512 tokens over 16,384 keys in a table of 512 rows 1,134 / 3,986 us.
constexpr int64_t kFewGridAlone = 1 << 20;
// Fewer beside prompts, where all may find nothing: 64 requests of up to 8,192 keys with
// 12 tokens each 228 / 224 us (without this launch 215), with 32 260 / 256 (248), with 2
// 151 / 153, 63 single tokens and a prompt of 512 185 / 185.  (4,096: 221, 253, 157, 189.)
constexpr int64_t kFewGridBeside = 8192;

int64_t few_spans(const KvWeighArgs& a) {
  const int64_t most = a.prompts && !idle_rows(a)   ? kFewGridBeside
                       : a.prompts || !some_many(a) ? kFewGrid
                                                    : kFewGridAlone;
  const int64_t rows = std::max<int64_t>(1, a.q.requests * a.c.heads);
  return std::min(chunks_of(a, kSpan, a.longest), std::max<int64_t>(1, most / rows));
}
int64_t few_grid(const KvWeighArgs& a) { return a.q.requests * a.c.heads * few_spans(a); }
int64_t prompts_grid(const KvWeighArgs& a) {
  return std::min(a.most_units, std::max<int64_t>(1, kGrid / a.c.heads)) * a.c.heads;
}

template <int DP, bool BF16>
void launch_dim(const KvWeighArgs& a, hipStream_t s) {
  if (a.prompts) kv_weigh_kernel<DP, BF16><<<dim3((unsigned)prompts_grid(a)), 256, 0, s>>>(a);
  if (a.few_rows > 0)
    kv_weigh_few_kernel<DP, BF16>
        <<<dim3((unsigned)few_grid(a)), 256, 0, s>>>(a, (int)few_spans(a));
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
  // (the kernel of prompts reads some key in place of an absent one: there has to be one)
  a.prompts = a.q.tokens > 0 && a.q.cols > 0 && a.q.group <= kRows && a.c.pages > 0 &&
              (!idle_rows(a) || (some_many(a) && a.q.requests <= kDealtRequests && room_of(a) >= kDealt));
  a.few_rows = !a.prompts                                      ? INT64_MAX
               : idle_rows(a) || a.q.requests >= kSomeRequests ? few_rows_of(a)
                                                               : 0;
  a.most_units = a.most_several = a.most_slots = 0;
  if (!a.prompts) return;
  a.tile = kRows / a.q.group;
  // a chunk of several units has two for each one more than the first, at most
  const int64_t extra = more_units(a);
  a.most_units = chunks_of(a, kChunk, INT32_MAX) * a.q.requests + extra;
  a.most_several = extra;
  a.most_slots = 2 * extra;
}

int64_t kv_weigh_workspace(const KvWeighArgs& a) {
  if (!a.prompts) return 0;
  return 4 * header_ints(a) + (a.most_units + a.most_several) * (int64_t)sizeof(Unit) +
         a.most_slots * a.c.heads * kChunk * 4;
}

int64_t kv_weigh_grid(const KvWeighArgs& a) {
  return std::max(a.few_rows > 0 ? few_grid(a) : 0, a.prompts ? prompts_grid(a) : 0);
}

hipError_t launch_kv_weigh(const KvWeighArgs& a, hipStream_t s) {
  if (a.prompts) {
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
