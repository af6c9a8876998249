// The best blocks of a paged cache for every new token: a cheap score of each
// block's summary, and the n best by it.
//
// The query of a (token, kv head): each value of its group's heads over the
// largest of all of them in 127ths, rounded to whole numbers; their sums over
// the heads; the sums in 127ths of the largest.  A block's score is the exact
// int8 dot product of that with the summary's codes, in float32 (below 2^24:
// exact), times the summary's scale.  So the order of the blocks is a matter of
// definition and not of rounding: every split, tile or kernel lists the same
// blocks.  Candidates are the complete blocks before the token's own; its own,
// the latest and the first ones are always taken.
//
// Ranks are 32-bit keys in the scores' order: 0 for no candidate, all ones for
// a block that is always taken.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>

#include "kv_cache.h"
#include "kv_values.h"

namespace mlxvs::kern {
namespace {

typedef uint32_t uintx2 __attribute__((ext_vector_type(2)));

constexpr uint32_t kAlways = 0xFFFFFFFFu;
constexpr int kLdsCols = 8192;  // ranks of a row that stay in LDS (32 KB)

// Bits set, signed: counts are subtracted and compared.
__device__ __forceinline__ int bits(uint64_t x) { return (int)__popcll(x); }

__device__ __forceinline__ uint32_t rank_of(int dot, float scale) {
  // a summary that is not finite ranks first (a broken block is not left out)
  float x = fabsf(scale) < __builtin_inff() ? (float)dot * scale : FLT_MAX;
  x = fminf(fmaxf(x, -FLT_MAX), FLT_MAX) + 0.0f;  // (-0 and 0 are equal)
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  return u >> 31 ? ~u : u | 0x80000000u;
}

// |x|, infinity for what is not finite (a NaN would get lost in a maximum).
__device__ __forceinline__ float finite_abs(float x) {
  x = fabsf(x);
  return x < __builtin_inff() ? x : __builtin_inff();
}
// The factor that takes values of at most `top` to codes, 0 where there is none.
__device__ __forceinline__ float to_codes(float top) {
  return top > 1e-30f && top < __builtin_inff() ? 127.0f / top : 0.0f;
}

// The codes of a (token, head)'s query, zeros past dim.  A query that holds
// nothing, or a value that is not finite, has codes 0.
template <bool BF16, int THREADS>
__device__ void query_codes(const KvSelectArgs& a, int64_t t, int h, int8_t* codes,
                            float* shared) {
  const int d = threadIdx.x, g = a.q.group;
  const uint16_t* q = (const uint16_t*)a.q.q + t * a.q.q_token + (int64_t)h * g * a.q.q_head + d;
  float top = 0.0f;
  if (d < a.c.dim) {
#pragma unroll 8
    for (int i = 0; i < g; ++i) top = fmaxf(top, finite_abs(value<BF16>(q[i * a.q.q_head])));
  }
  top = block_max<THREADS>(top, shared);
  const float inv = to_codes(top);
  int sum = 0;
  if (d < a.c.dim && inv != 0.0f) {
#pragma unroll 8
    for (int i = 0; i < g; ++i) sum += (int)rintf(value<BF16>(q[i * a.q.q_head]) * inv);
  }
  const float peak = block_max<THREADS>((float)abs(sum), shared);
  const float to = peak > 0.0f ? 127.0f / peak : 0.0f;
  if (d < kKvMaxDim) codes[d] = (int8_t)rintf((float)sum * to);
  __syncthreads();
}

typedef int intx4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ intx4 mfma_i8(uintx4 x, uintx4 y, intx4 c) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(intx4, x),
                                               __builtin_bit_cast(intx4, y), c, 0, 0, 0);
#else
  return c;
#endif
}

// query_codes of a wavefront's tokens t0, t0 + step, ..: two neighbouring values
// a lane (KD / 128 times), the loads of all tokens and eight heads in flight.
template <bool BF16, int KD, int NT>
__device__ void wave_query_codes(const KvSelectArgs& a, int64_t t0, int step, int h,
                                 int8_t* codes, int stride) {
  constexpr int P = (KD + 127) / 128, HEADS = 8;
  const int lane = threadIdx.x & 63, g = a.q.group;
  const uint16_t* q[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
    q[t] = (const uint16_t*)a.q.q + min(t0 + t * step, a.q.tokens - 1) * a.q.q_token +
           (int64_t)h * g * a.q.q_head;
  const auto each = [&](auto&& f) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int d = 2 * (lane + 64 * p);
      if (d >= a.c.dim) continue;
      for (int i0 = 0; i0 < g; i0 += HEADS) {
        uint32_t x[NT][HEADS];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < HEADS; ++i)  // (past the last head: zeros, which add nothing)
            x[t][i] = i0 + i < g ? *(const uint32_t*)(q[t] + (i0 + i) * a.q.q_head + d) : 0;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < HEADS; ++i)
            f(t, p, value<BF16>((uint16_t)x[t][i]), value<BF16>((uint16_t)(x[t][i] >> 16)));
      }
    }
  };
  float inv[NT] = {}, peak[NT] = {};
  int s0[NT][P] = {}, s1[NT][P] = {};
  each([&](int t, int, float u, float v) {
    inv[t] = fmaxf(inv[t], fmaxf(finite_abs(u), finite_abs(v)));
  });
#pragma unroll
  for (int t = 0; t < NT; ++t) inv[t] = to_codes(wave_max(inv[t]));
  each([&](int t, int p, float u, float v) {
    // (a factor of 0 belongs to values that may not be finite)
    s0[t][p] += inv[t] != 0.0f ? (int)rintf(u * inv[t]) : 0;
    s1[t][p] += inv[t] != 0.0f ? (int)rintf(v * inv[t]) : 0;
  });
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int p = 0; p < P; ++p)
      peak[t] = fmaxf(peak[t], fmaxf((float)abs(s0[t][p]), (float)abs(s1[t][p])));
    peak[t] = wave_max(peak[t]);
    const float to = peak[t] > 0.0f ? 127.0f / peak[t] : 0.0f;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int d = 2 * (lane + 64 * p);
      if (d < KD) {
        const int x = (int)rintf((float)s0[t][p] * to), y = (int)rintf((float)s1[t][p] * to);
        *(uint16_t*)(codes + t * step * stride + d) = (uint16_t)((x & 255) | (y & 255) << 8);
      }
    }
  }
}

// Scores of 16 columns' blocks a step, by one wavefront: their summaries are the
// rows of the 16x16x64 int8 MFMA (lane l: 16 bytes of the block of column l %
// 16), the codes of 16 queries, or one sixteen times, its columns.  KD: head
// size rounded up to a multiple of 64.  A16: rows of summaries are 16-byte
// aligned (else 8).  AHEAD steps are in flight at a time, each `stride` columns
// and `heads` heads past the one before; those from `steps` on are empty.
template <int KD, bool A16, int AHEAD>
struct BlockScores {
  uintx4 v[AHEAD][KD / 64];
  float scale[AHEAD];
  uint32_t present[AHEAD];  // bit m: column m of the step has a page

  __device__ __forceinline__ void load(const KvSelectArgs& a, int h, const int32_t* table, int j0,
                                       int stride, int count, int heads = 0, int steps = AHEAD) {
    const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
    int p[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int j = j0 + u * stride + col;
      p[u] = j < count && u < steps ? table[j] : -1;
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const bool there = p[u] >= 0 && p[u] < a.c.pages;
      const int64_t row = (int64_t)p[u] * a.c.heads + h + u * heads;
      const int8_t* m = a.c.summaries + row * a.c.dim;
      scale[u] = 0.0f;
      if (there) scale[u] = a.c.scales[row];
#pragma unroll
      for (int i = 0; i < KD / 64; ++i) {
        const int at = 64 * i + 16 * grp;
        v[u][i] = uintx4{};
        if constexpr (A16) {
          if (there && at < a.c.dim) v[u][i] = *(const uintx4*)(m + at);
        } else {
          if (there && at < a.c.dim) *(uintx2*)&v[u][i] = *(const uintx2*)(m + at);
          if (there && at + 8 < a.c.dim) *((uintx2*)&v[u][i] + 1) = *(const uintx2*)(m + at + 8);
        }
      }
      present[u] = (uint32_t)__ballot(there);
    }
  }

  // The ranks of step u under one query, its codes in all 16 columns: columns j0
  // .. of a row of `count`, up to the block `own`.
  __device__ __forceinline__ void put(const KvSelectArgs& a, int u, const uintx4 (&codes)[KD / 64],
                                      int own, int j0, int count, uint32_t* ranks) const {
    const intx4 d = dots(u, codes);
    // the 16 columns of the product are alike: lane l ranks row 4 grp + l % 4
    const int lane = threadIdx.x & 63, i = lane & 3, m = 4 * (lane >> 4) + i, j = j0 + m;
    const float s = __shfl(scale[u], m);
    const int dot = i & 2 ? (i & 1 ? d[3] : d[2]) : (i & 1 ? d[1] : d[0]);
    if ((lane & 15) < 4 && j < count)
      ranks[j] = !(present[u] >> m & 1)              ? 0
                 : j < a.first || j > own - a.last ? kAlways
                                                     : rank_of(dot, s);
  }

  // Row 4 grp + i of step u: its dot product with the lane's column of codes.
  __device__ __forceinline__ intx4 dots(int u, const uintx4 (&codes)[KD / 64]) const {
    intx4 d = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < KD / 64; ++i) d = mfma_i8(v[u][i], codes[i], d);
    return d;
  }
};

template <int KD>
__device__ __forceinline__ void load_codes(uintx4 (&q)[KD / 64], const int8_t* codes) {
#pragma unroll
  for (int i = 0; i < KD / 64; ++i)
    q[i] = *(const uintx4*)(codes + 64 * i + 16 * ((threadIdx.x & 63) >> 4));
}

// Ranks of the columns [0, count) of one query into LDS.  make() leaves its
// codes in `codes` (it waits for the workgroup) while the first summaries are
// on their way.
template <int KD, bool A16, int AHEAD, int THREADS, typename Make>
__device__ void rank_row(const KvSelectArgs& a, int h, int own, const int32_t* table, int count,
                         const int8_t* codes, uint32_t* ranks, Make make) {
  constexpr int STRIDE = 16 * (THREADS / 64);
  int j0 = 16 * __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  BlockScores<KD, A16, AHEAD> b;
  b.load(a, h, table, j0, STRIDE, count);
  make();
  uintx4 q[KD / 64];
  load_codes<KD>(q, codes);
  while (j0 < count) {
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) b.put(a, u, q, own, j0 + u * STRIDE, count, ranks);
    j0 += AHEAD * STRIDE;
    if (j0 < count) b.load(a, h, table, j0, STRIDE, count);
  }
}

// Of a wavefront's N x 64 ranks: a `cut` that n of them reach (`upto` == n), or
// the n-th largest, which more do; bit by bit, counting with ballots: no barrier.
// Fewer than n candidates: 0.
struct Cut {
  uint32_t cut;
  int upto;
};

template <int N>
__device__ __forceinline__ Cut wave_cut(const uint32_t (&k)[N], int n) {
  Cut r{0, 0};
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t c = r.cut | 1u << bit;
    int m = 0;
#pragma unroll
    for (int x = 0; x < N; ++x) m += bits(__ballot(k[x] >= c));
    if (m >= n) {
      r = {c, m};
      if (m == n) break;
    }
  }
  return r;
}

template <int N>
__device__ __forceinline__ int wave_above(const uint32_t (&k)[N], uint32_t cut) {
  int m = 0;
#pragma unroll
  for (int x = 0; x < N; ++x) m += bits(__ballot(k[x] > cut));
  return m;
}

// The n largest of a row's ranks in LDS by one wavefront (lane l: 64 x + l), the
// lowest columns among equal ones, ascending by column into out, -1 after.  The
// row is written over.
//
// A cut of the lanes' largest ranks is one that at least n of all reach, and few
// more (64 ln(64 / (64 - n)) if they lie at random: 18 for 16, 44 for 32): those
// are gathered, one a lane, and cut again, so that a count is one ballot and not
// NR.  2,048 rows, n = 16, with NR ballots a count / so: 20.7 / 17.5 us at 512
// columns, 29.3 / 21.6 at 891, 47.5 / 28.0 at 1,024, 53.3 / 33.8 at 2,048; n = 64,
// of which more reach than there are lanes: 54.4 / 56.6 at 2,048.
constexpr int kGather = 32;  // the longest lists made so

template <int NR>
__device__ void wave_take_best(uint32_t* ranks, int count, int n, int32_t* out) {
  const int lane = threadIdx.x & 63;
  const uint64_t below = (uint64_t(1) << lane) - 1;
  uint32_t k[NR], top[1] = {0};
#pragma unroll
  for (int x = 0; x < NR; ++x) {
    k[x] = 64 * x + lane < count ? ranks[64 * x + lane] : 0;
    top[0] = max(top[0], k[x]);
  }
  // all ranks from `cut` on are taken, of those equal to it the first `ties`
  uint32_t cut = 1;
  int ties = 64 * NR;
  if (count > n) {
    Cut c = n <= kGather ? wave_cut(top, n) : Cut{0, 0};
    const int reach = c.cut ? wave_above(k, c.cut - 1) : 0;
    if (reach == n) {
      cut = c.cut;
    } else if (reach > n && reach <= 64) {
      int at = 0;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (int x = 0; x < NR; ++x) {
        const uint64_t some = __ballot(k[x] >= c.cut);
        if (k[x] >= c.cut) ranks[at + bits(some & below)] = k[x];
        at += bits(some);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      const uint32_t few[1] = {lane < reach ? ranks[lane] : 0};
      c = wave_cut(few, n);
      cut = c.cut;
      if (c.upto > n) ties = n - wave_above(few, cut);
    } else {
      // longer lists, blocks that are absent from many lanes, or many equal ranks
      c = wave_cut(k, n);
      if (c.cut) cut = c.cut;  // (else fewer candidates than n: all)
      if (c.upto > n) ties = n - wave_above(k, cut);
    }
  }
  int at = 0;
#pragma unroll
  for (int x = 0; x < NR; ++x) {
    const uint64_t tied = __ballot(k[x] == cut);
    const bool take = k[x] > cut || (k[x] == cut && bits(tied & below) < ties);
    const uint64_t taken = __ballot(take);
    if (take) out[at + bits(taken & below)] = 64 * x + lane;
    at += bits(taken);
    ties -= bits(tied);
  }
  for (int x = at + lane; x < n; x += 64) out[x] = -1;
}

template <int THREADS>
struct Select {
  uint32_t hist[256];
  int gt[THREADS / 64], eq[THREADS / 64];
  uint32_t prefix;
  int left;
};

// The n largest of ranks[0 .. count), the lowest columns among equal ones,
// ascending by column into out, -1 after.
template <int THREADS>
__device__ void take_best(const uint32_t* ranks, int count, int n, int32_t* out,
                          Select<THREADS>& s) {
  constexpr int kWaves = THREADS / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // the n-th largest rank, 8 bits at a time
  uint32_t prefix = 0;
  int left = n;
  if (count > n) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (threadIdx.x < 256) s.hist[threadIdx.x] = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < count; i += THREADS) {
        const uint32_t k = ranks[i];
        if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8)))
          atomicAdd(&s.hist[(k >> shift) & 255], 1u);
      }
      __syncthreads();
      if (wave == 0) {
        // lane l: bins 4 l .. 4 l + 3, counted from the top
        int c[4], sum = 0;
#pragma unroll
        for (int i = 3; i >= 0; --i) c[i] = sum += (int)s.hist[4 * lane + i];
        int above = sum;
#pragma unroll
        for (int x = 1; x < 64; x *= 2) {
          const int y = __shfl_down(above, x);
          if (lane + x < 64) above += y;
        }
        above -= sum;  // in the bins of the lanes past this one
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int upto = above + c[i], before = i < 3 ? above + c[i + 1] : above;
          if (before < left && upto >= left) {
            s.prefix = prefix | (uint32_t)(4 * lane + i) << shift;
            s.left = left - before;
          }
        }
      }
      __syncthreads();
      prefix = s.prefix;
      left = s.left;
    }
  }
  // each wavefront a stretch of the columns: those above the n-th, and the
  // first `left` that equal it (all that are candidates, if they are few)
  const bool few = count <= n;
  const int per = (count + kWaves * 64 - 1) / (kWaves * 64) * 64;
  const int from = wave * per, to = min(count, from + per);
  int gt = 0, eq = 0;
  for (int i = from + lane; i - lane < to; i += 64) {
    const uint32_t k = i < to ? ranks[i] : 0;
    gt += bits(__ballot(few ? k > 0 : k > prefix));
    if (!few) eq += bits(__ballot(i < to && k == prefix && k > 0));
  }
  if (lane == 0) {
    s.gt[wave] = gt;
    s.eq[wave] = eq;
  }
  __syncthreads();
  int at = 0, ties = 0;
  for (int w = 0; w < wave; ++w) {
    at += s.gt[w] + min(s.eq[w], max(0, left - ties));
    ties += s.eq[w];
  }
  const uint64_t below = (uint64_t(1) << lane) - 1;
  for (int i = from + lane; i - lane < to; i += 64) {
    const uint32_t k = i < to ? ranks[i] : 0;
    const bool up = few ? k > 0 : k > prefix, tie = !few && i < to && k == prefix && k > 0;
    const uint64_t tied = __ballot(tie);
    const bool take = up || (tie && ties + bits(tied & below) < left);
    const uint64_t taken = __ballot(take);
    if (take) out[at + bits(taken & below)] = i;
    at += bits(taken);
    ties += bits(tied);
  }
  int all = 0, tied = 0;
  for (int w = 0; w < kWaves; ++w) {
    all += s.gt[w];
    tied += s.eq[w];
  }
  all += min(tied, left);
  for (int i = all + threadIdx.x; i < n; i += THREADS) out[i] = -1;
}

// Columns of a row that may be listed: up to its own block's.
__device__ __forceinline__ int columns_of(const KvSelectArgs& a, int64_t t, int* r, int* own) {
  *r = a.q.token_request[t];
  const int pos = a.q.positions[t];
  *own = pos >= 0 ? pos >> a.c.lps : -1;
  return *r >= 0 && *r < a.q.requests ? min(*own + 1, a.q.cols) : 0;
}

// Steps in flight (registers: 16 bytes a step and 64 values).
constexpr int ahead(int kd) { return kd == 256 ? 4 : 8; }

// A row's ranks in LDS, then its list.
template <bool BF16, int KD, bool A16, int THREADS>
__global__ __launch_bounds__(THREADS) void kv_select_kernel(KvSelectArgs a) {
  extern __shared__ uint32_t ranks[];
  __shared__ Select<THREADS> s;
  __shared__ __align__(16) int8_t codes[kKvMaxDim];
  __shared__ float red[THREADS / 64];
  const int h = (int)(blockIdx.x % a.c.heads);
  const int64_t t = blockIdx.x / a.c.heads;
  int r, own;
  const int count = columns_of(a, t, &r, &own);
  const int32_t* table = a.q.table + (int64_t)r * a.q.table_stride;
  if (count > a.n) {  // (else every candidate is taken, whatever its score)
    rank_row<KD, A16, ahead(KD), THREADS>(
        a, h, own, table, count, codes, ranks,
        [&] { query_codes<BF16, THREADS>(a, t, h, codes, red); });
  } else {
    for (int j = threadIdx.x; j < count; j += THREADS) {
      const int p = table[j];
      ranks[j] = p >= 0 && p < a.c.pages ? kAlways : 0;
    }
  }
  __syncthreads();
  take_best(ranks, count, a.n, a.blocks + (t * a.c.heads + h) * a.n, s);
}

// Long rows: ranks to the workspace, 128 columns of up to 8 heads a workgroup
// (a page's summaries and scales lie side by side over its heads), 16 columns a
// wavefront ...
constexpr int kPartCols = 128, kPartHeads = 8;

template <bool BF16, int KD, bool A16>
__global__ __launch_bounds__(512) void kv_select_ranks_kernel(KvSelectArgs a, int parts) {
  __shared__ __align__(16) int8_t codes[kPartHeads][KD + 16];
  const int part = (int)(blockIdx.x % parts);
  const int sets = (a.c.heads + kPartHeads - 1) / kPartHeads;
  const int h0 = (int)(blockIdx.x / parts % sets) * kPartHeads;
  const int64_t t = blockIdx.x / parts / sets;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int heads = min(kPartHeads, a.c.heads - h0);
  int r, own;
  const int count = columns_of(a, t, &r, &own);
  if (part * kPartCols >= count) return;
  const int j0 = part * kPartCols + 16 * wave;
  BlockScores<KD, A16, kPartHeads> b;
  b.load(a, h0, a.q.table + (int64_t)r * a.q.table_stride, j0, 0, count, 1, heads);
  if (wave < heads) wave_query_codes<BF16, KD, 1>(a, t, 0, h0 + wave, codes[wave], 0);
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kPartHeads; ++u) {
    if (u >= heads) break;
    uintx4 q[KD / 64];
    load_codes<KD>(q, codes[u]);
    b.put(a, u, q, own, j0, count, a.keys + (t * a.c.heads + h0 + u) * a.q.cols);
  }
}

// ... and the lists from there, by way of LDS if they fit.
__global__ __launch_bounds__(1024) void kv_select_lists_kernel(KvSelectArgs a, bool lds) {
  extern __shared__ uint32_t held[];
  __shared__ Select<1024> s;
  const int64_t row = blockIdx.x;
  int r, own;
  const int count = columns_of(a, row / a.c.heads, &r, &own);
  const uint32_t* ranks = a.keys + row * a.q.cols;
  if (lds) {
#pragma unroll 8
    for (int i = threadIdx.x; i < count; i += 1024) held[i] = ranks[i];
    __syncthreads();
  }
  take_best(lds ? held : ranks, count, a.n, a.blocks + row * a.n, s);
}

// Prompts: 16 tokens and a head a workgroup.  Scores are an int8 product of 16
// blocks' summaries and the 16 tokens' codes on the 16x16x64 MFMA, ranks go to
// LDS, and each wavefront lists the best of 2 tokens.  NR: ranks a lane holds.
constexpr int kTile = 16;

template <bool BF16, int KD, bool A16, int NR>
__global__ __launch_bounds__(512) void kv_select_tile_kernel(KvSelectArgs a) {
  constexpr int W = 8, S = 64 * NR + 4;  // (rows 4 banks apart)
  constexpr int AHEAD = KD == 256 ? 2 : 4;
  extern __shared__ __align__(16) uint32_t ranks[];  // [kTile][S]
  __shared__ __align__(16) int8_t codes[kTile][KD + 16];
  __shared__ int req[kTile], cnt[kTile], own[kTile];
  const int h = (int)(blockIdx.x % a.c.heads);
  const int64_t t0 = (int64_t)(blockIdx.x / a.c.heads) * kTile;
  const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (threadIdx.x < kTile) {
    int r = -1, o = -1, n = 0;
    if (t0 + threadIdx.x < a.q.tokens) n = columns_of(a, t0 + threadIdx.x, &r, &o);
    req[threadIdx.x] = r;
    own[threadIdx.x] = o;
    cnt[threadIdx.x] = n;
  }
  wave_query_codes<BF16, KD, kTile / W>(a, t0 + wave, W, h, codes[wave], KD + 16);
  __syncthreads();
  uintx4 q[KD / 64];
  load_codes<KD>(q, codes[col]);
  const int myreq = req[col], mycnt = cnt[col], myown = own[col];
  // the requests of the tile one after another (most often there is one)
  for (uint64_t todo = __ballot(mycnt > 0) & 0xFFFF; todo;) {
    const int r = __builtin_amdgcn_readlane(myreq, __builtin_ctzll(todo));
    const bool mine = mycnt > 0 && myreq == r;
    int most = mine ? mycnt : 0;
#pragma unroll
    for (int x = 1; x < 16; x *= 2) most = max(most, __shfl_xor(most, x));
    todo &= ~__ballot(mine);
    const int32_t* table = a.q.table + (int64_t)r * a.q.table_stride;
    for (int j0 = 16 * wave; j0 < most; j0 += 16 * W * AHEAD) {
      BlockScores<KD, A16, AHEAD> b;
      b.load(a, h, table, j0, 16 * W, most);
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const intx4 d = b.dots(u, q);
        uintx4 k;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int m = 4 * grp + i, j = j0 + 16 * W * u + m;
          const float s = __shfl(b.scale[u], m);
          k[i] = !(b.present[u] >> m & 1)              ? 0
                 : j < a.first || j > myown - a.last ? kAlways
                                                       : rank_of(d[i], s);
        }
        const int j = j0 + 16 * W * u + 4 * grp;
        if (mine && j < 64 * NR) *(uintx4*)&ranks[col * S + j] = k;
      }
    }
  }
  __syncthreads();
  for (int i = wave; i < kTile && t0 + i < a.q.tokens; i += W)
    wave_take_best<NR>(ranks + i * S, cnt[i], a.n, a.blocks + ((t0 + i) * a.c.heads + h) * a.n);
}

// Ways to list (rows: tokens x kv heads; figures for 128 values, 4 heads a kv head):
// - kTile, 16 tokens a workgroup, where requests have many: a block is read once
//   for 16 tokens, but a launch is no shorter than a workgroup.  By row / by tile,
//   16 blocks taken: 1,024 rows of one request 10.4 / 10.0 us at 64 columns, 20.4 /
//   17.4 at 512, 28.0 / 21.6 at 891, 30.2 / 27.9 at 1,024 (a workgroup has a CU to
//   itself from 897 on), 52.2 / 33.6 at 2,048; 2,048 rows 18.5 / 10.1, 35.8 / 17.1,
//   48.8 / 21.9, 53.4 / 28.0, 92.9 / 33.7; 768 rows 9.7 / 11.7 at 64, 17.7 / 17.0 at
//   512, 26.1 / 27.3 at 1,024.  32 requests of 8 tokens 35.8 / 20.6, 16 requests of 8
//   20.2 / 20.4.  64 taken of 2,048 columns: 2,048 rows 55 by tile, as long as 1,024
//   rows by row.
// - kRow, a row a workgroup, its ranks in LDS.
// - kParts, two launches over the workspace, for a few long rows (or ranks that no
//   LDS holds): by row / in two launches, 128 rows 21.0 / 18.6 us at 2,048 columns,
//   31.5 / 26.0 at 4,096; 8 rows 14.4 / 16.6 at 1,024; 256 rows 22.3 / 24.1 at
//   2,048, 31.8 / 37.1 at 4,096.
// Beyond kTileCols columns prompts go by rows too, each reading its summaries again:
// 1,500 tokens of 8 heads 99 us at 2,048 columns, 490 at 2,049, 1,725 at 8,192.  "Many"
// tokens go by the table's height, idle rows included: 512 tokens of 8 heads over 512
// columns 17 us, 64 in a table of 256 rows.
// What bounds small calls is a chain of five dependent accesses, about 10 us
// whatever the size; large ones, the listing (32 counts of a row's ranks).
enum class Way { kRow, kParts, kTile };

constexpr int kTileCols = 64 * 32;  // ranks of 16 tokens in 128 KB of LDS

Way way_of(const KvSelectArgs& a) {
  const int64_t rows = a.q.tokens * a.c.heads;
  const int64_t many = a.q.cols <= 896 || a.n <= kGather ? 1024 : 1536;
  if (a.q.cols <= kTileCols && rows >= many && a.q.tokens >= 8 * a.q.requests) return Way::kTile;
  return a.q.cols > kLdsCols || (a.q.cols > 1024 && rows < 256) ? Way::kParts : Way::kRow;
}

template <bool BF16, int KD, bool A16, int NR>
void launch_tile(const KvSelectArgs& a, hipStream_t s) {
  const unsigned grid = (unsigned)((a.q.tokens + kTile - 1) / kTile * a.c.heads);
  kv_select_tile_kernel<BF16, KD, A16, NR><<<grid, 512, kTile * (64 * NR + 4) * 4, s>>>(a);
}

template <bool BF16, int KD, bool A16>
void launch_select(const KvSelectArgs& a, hipStream_t s) {
  const unsigned rows = (unsigned)(a.q.tokens * a.c.heads);
  switch (way_of(a)) {
    case Way::kTile:
      if (a.q.cols <= 256) launch_tile<BF16, KD, A16, 4>(a, s);
      else if (a.q.cols <= 512) launch_tile<BF16, KD, A16, 8>(a, s);
      else if (a.q.cols <= 896) launch_tile<BF16, KD, A16, 14>(a, s);
      else launch_tile<BF16, KD, A16, 32>(a, s);
      return;
    case Way::kRow:
      // (1,024 / 256 threads: 256 rows 15.2 / 18.0 us at 1,024 columns, 10.4 / 10.1
      // at 256; 384 rows 26.1 / 23.0 and 18.9 / 10.4)
      if (rows <= 256 && a.q.cols > 512)
        kv_select_kernel<BF16, KD, A16, 1024><<<rows, 1024, a.q.cols * 4, s>>>(a);
      else kv_select_kernel<BF16, KD, A16, 256><<<rows, 256, a.q.cols * 4, s>>>(a);
      return;
    case Way::kParts:
      const int parts = (a.q.cols + kPartCols - 1) / kPartCols;
      const int sets = (a.c.heads + kPartHeads - 1) / kPartHeads;
      const bool lds = a.q.cols <= kLdsCols;
      kv_select_ranks_kernel<BF16, KD, A16>
          <<<(unsigned)(a.q.tokens * sets * parts), 512, 0, s>>>(a, parts);
      kv_select_lists_kernel<<<rows, 1024, lds ? a.q.cols * 4 : 0, s>>>(a, lds);
  }
}

template <bool BF16>
void launch_dim(const KvSelectArgs& a, hipStream_t s) {
  const bool a16 = a.c.dim % 16 == 0;
  if (a.c.dim <= 64) a16 ? launch_select<BF16, 64, true>(a, s) : launch_select<BF16, 64, false>(a, s);
  else if (a.c.dim <= 128) a16 ? launch_select<BF16, 128, true>(a, s) : launch_select<BF16, 128, false>(a, s);
  else a16 ? launch_select<BF16, 256, true>(a, s) : launch_select<BF16, 256, false>(a, s);
}

}  // namespace

int64_t kv_select_workspace(const KvSelectArgs& a) {
  return way_of(a) == Way::kParts ? a.q.tokens * a.c.heads * a.q.cols * 4 : 0;
}

int64_t kv_select_grid(const KvSelectArgs& a) {
  // (in workgroups of 256)
  const int64_t rows = a.q.tokens * a.c.heads;
  switch (way_of(a)) {
    case Way::kTile: return 2 * ((a.q.tokens + kTile - 1) / kTile * a.c.heads);
    case Way::kRow: return rows <= 256 ? 4 * rows : rows;
    case Way::kParts: break;
  }
  const int64_t parts = (a.q.cols + kPartCols - 1) / kPartCols;
  const int64_t sets = (a.c.heads + kPartHeads - 1) / kPartHeads;
  return std::max(2 * a.q.tokens * sets * parts, 4 * rows);
}

hipError_t launch_kv_select(const KvSelectArgs& a, hipStream_t s) {
  a.c.bf16 ? launch_dim<true>(a, s) : launch_dim<false>(a, s);
  return hipGetLastError();
}

}  // namespace mlxvs::kern
