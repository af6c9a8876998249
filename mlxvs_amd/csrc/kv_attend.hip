// Attention of new tokens over the paged key-value cache: over every block up
// to the token's position, or over the blocks of a list of its own.
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - max)
//
// over the keys j that the token sees, one pass with the running maximum and
// sum.  The G query heads of a kv head are the 16 columns of the products:
// S^T = K Q^T and O^T = V^T P^T, both on the 16x16x32 MFMA (bf16 / f16 in,
// float32 out).  With values transposed within a page, K rows and V^T rows are
// 16-byte loads in the A operand's own layout: a single token's go from the cache
// straight into registers (those of prompts, which share them, through LDS); and
// S^T comes out with its keys along the registers.  The keys of a 32-key pair
// of S tiles are dealt to the tiles' rows so that a lane ends up with 8
// consecutive keys (row m of tile t is key 8 (m / 4) + 4 t + m % 4): exactly
// the 8 keys it holds of the second product's B operand, so P stays in its
// registers too, and the V^T loads stay 16 bytes wide.
//
// P is rounded to the cache's type for the second product (the values' own
// precision; a sum of roundings that averages out: error against 64 bits 2.0e-3 of
// an output's norm in bf16 and 2.5e-4 in f16, where the output's own rounding makes
// 1.7e-3 and 2.1e-4), its sum is not; under f16 P is scaled up, by 2^14 or, for
// prompts, 2^7, so that small terms of long sums stay normal numbers.
// Scores, maxima, sums and the output are float32.
//
// Single tokens are bound by HBM: 64 ragged requests of up to 8,192 tokens (8 kv
// heads of 4, 128 values) 247 us, 4.9 TB/s; one of 262,144 188 us, 5.7 TB/s (a large
// read alone: 6.3 TB/s with plain loads).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "kv_cache.h"
#include "kv_lists.h"
#include "lds_stage.h"

namespace mlxvs::kern {
namespace {

typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef _Float16 halfx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));

constexpr int kColumns = 16;  // query heads of one product
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ floatx4 mfma(bf16x8 a, bf16x8 b, floatx4 c) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
#else
  return c;
#endif
}
__device__ __forceinline__ floatx4 mfma(halfx8 a, halfx8 b, floatx4 c) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
#else
  return c;
#endif
}

// The maximum over the lanes of one column (l, l ^ 16, l ^ 32, l ^ 48).  The lane
// swaps are VALU instructions: a shuffle would wait for LDS.  (Written out: the
// builtins' two results are taken for one where both operands are one value.
// The instruction reads other lanes' registers two wait states after a write.)
__device__ __forceinline__ float column_max(float x) {
#if defined(__HIP_DEVICE_COMPILE__)
  float y = x;
  asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(x), "+v"(y));
  x = y = fmaxf(x, y);
  asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(x), "+v"(y));
  x = fmaxf(x, y);
#endif
  return x;
}
__device__ __forceinline__ float column_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// An entry of a block table, by a scalar load: the same for a whole wavefront, and
// not written while the kernel runs.
__device__ __forceinline__ int table_entry(const int32_t* table, int i) {
  return *(const __attribute__((address_space(4))) int32_t*)(uintptr_t)(table + i);
}

// A token's position, at most the table's last (-1 for a table without columns):
// beyond it there is nothing to see, and position + 1 fits in 31 bits.
__device__ __forceinline__ int position(const KvAttendArgs& a, int64_t t) {
  return min(a.q.positions[t], (a.q.cols << a.c.lps) - 1);
}

// The first `n` of 8 values (n <= 0: none), zeros after.
__device__ __forceinline__ uintx4 keep(uintx4 v, int n) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = n - 2 * i;
    v[i] &= m >= 2 ? 0xFFFFFFFFu : (m == 1 ? 0xFFFFu : 0u);
  }
  return v;
}

// Head sizes are rounded up to one of these; a kernel for DP has more values than
// the next smaller one holds, so that only the last of them need a check.
constexpr int kSizes[] = {64, 96, 128, 192, 256};
constexpr int sure_values(int dp) {
  int below = 0;
  for (int s : kSizes)
    if (s < dp) below = s;
  return below;
}

// log2 of what weights are scaled by: under f16 small terms of long sums stay
// normal numbers (the largest weight is 2^14).
template <typename T>
constexpr float kBiasOf = std::is_same_v<T, _Float16> ? 14.0f : 0.0f;

// The weights of a lane's scores, exp2(c s + bias - c max) rounded to T,
// with the running maximum m and this lane's sum l of its column, and the
// column's sums o scaled where the maximum moves.  (Letting the maximum lag by up
// to 2^8 spares most of that: 3% on prompts; but then the largest weights, which
// are whole otherwise, get rounded too: error against 64 bits 2.2e-3, not 2.0e-3.)
template <int S, int TILES, typename T8>
__device__ __forceinline__ void weights(floatx4 (&s)[2 * S], float& m, float& l, float c, float bias,
                                        floatx4 (&o)[TILES], T8 (&p)[S]) {
  using T = std::conditional_t<std::is_same_v<T8, bf16x8>, __bf16, _Float16>;
  float top = m;
#pragma unroll
  for (int u = 0; u < 2 * S; ++u)
#pragma unroll
    for (int i = 0; i < 4; ++i) top = fmaxf(top, s[u][i]);
  top = column_max(top);
  if (__any(top > m)) {
    const float w = top == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f((m - top) * c);
    l *= w;
#pragma unroll
    for (int i = 0; i < TILES; ++i) o[i] *= w;
    m = top;
  }
  const float low = bias - (m == -__builtin_inff() ? 0.0f : m) * c;
#pragma unroll
  for (int u = 0; u < S; ++u)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = __builtin_amdgcn_exp2f(fmaf(s[2 * u + i / 4][i % 4], c, low));
      l += x;
      p[u][i] = (T)x;
    }
}

// DP: head size rounded up.  LIST: over listed blocks.  P16: pages of 16 keys,
// two to a 32-key pair.
template <int DP, bool BF16, bool LIST, bool P16>
struct Attend {
  using T = std::conditional_t<BF16, __bf16, _Float16>;
  using Tx8 = std::conditional_t<BF16, bf16x8, halfx8>;
  using Tx4 = std::conditional_t<BF16, bf16x4, halfx4>;
  static constexpr int kChunks = DP / 32;           // k-steps of a score
  static constexpr int kTiles = DP / 16;            // rows of V^T
  static constexpr int kPairs = DP <= 128 ? 2 : 1;  // 32-key pairs a step
  static constexpr int kKeys = 32 * kPairs;
  static constexpr float kBias = kBiasOf<T>;

  const KvAttendArgs& a;
  const int lane, col, grp;
  const int d;         // values a head
  Tx8 q[kChunks];
  floatx4 o[kTiles];
  float m, l;          // running maximum of raw scores (of a column); this lane's sum
  float c;             // scale log2(e)

  // 64 entries of the row, one a lane: its page and how many of its keys show
  int page, seen;
  int e0;

  __device__ __forceinline__ Attend(const KvAttendArgs& args, int ln)
      : a(args), lane(ln), col(ln & 15), grp(ln >> 4), d(args.c.dim) {}

  __device__ __forceinline__ void start(int64_t t, int h, int mt) {
    const T* src = (const T*)a.q.q + t * a.q.q_token +
                   (int64_t)(h * a.q.group + mt * kColumns + col) * a.q.q_head;
    const bool mine = mt * kColumns + col < a.q.group;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int at = 32 * i + 8 * grp;
      uintx4 x = {};
      if (mine && at < d) x = *(const uintx4*)(src + at);
      q[i] = __builtin_bit_cast(Tx8, x);
    }
#pragma unroll
    for (int i = 0; i < kTiles; ++i) o[i] = floatx4{0, 0, 0, 0};
    m = -__builtin_inff();
    l = 0.0f;
    c = a.scale * kLog2e;
  }

  // Entries from `first` on of a row whose entries end at `end`.
  __device__ __forceinline__ void entries(int64_t t, int h, int r, int pos, int first, int end) {
    e0 = first;
    const int e = first + lane;
    page = 0;
    seen = 0;
    if (e < end) {
      int block = e;
      if constexpr (LIST) block = a.blocks[(t * a.c.heads + h) * a.n + e];
      if (block >= 0 && block < a.q.cols) {
        const int p = a.q.table[(int64_t)r * a.q.table_stride + block];
        // (block < cols, and cols pages fit in 31 bits)
        const int vis = pos + 1 - (block << a.c.lps);
        if (p >= 0 && p < a.c.pages && vis > 0) {
          page = p;
          seen = min(vis, a.c.page);
        }
      }
    }
  }

  // The step of kKeys keys from key `k` (of the row's listed keys) on.
  __device__ __forceinline__ void step(int h, int k) {
    const int ps = P16 ? 16 : a.c.page, lps = P16 ? 4 : a.c.lps;
    const int64_t head = (int64_t)ps * d;  // values of a (page, head)
    uintx4 kf[2 * kPairs][kChunks], vf[kPairs][kTiles];
    int n8[kPairs];  // of this lane's 8 keys of a pair, those that show
    bool all = true, any = false;
    const T* kp[kPairs];
    const T* vp[kPairs];
#pragma unroll
    for (int p = 0; p < kPairs; ++p) {
      const int kk = k + 32 * p;
      int pgK, pgV, sn;
      if constexpr (P16) {
        const int e = (kk >> 4) - e0;
        pgK = __shfl(page, e + (col >> 3));
        pgV = __shfl(page, e + (grp >> 1));
        sn = __shfl(seen, e + (grp >> 1));
      } else {
        const int e = (kk >> lps) - e0;
        pgK = pgV = __builtin_amdgcn_readlane(page, e);
        sn = __builtin_amdgcn_readlane(seen, e);
      }
      const int off = kk & (ps - 1);
      const int offK = P16 ? (8 * (col >> 2)) & 15 : off + 8 * (col >> 2);
      const int offV = P16 ? (8 * grp) & 15 : off + 8 * grp;
      kp[p] = (const T*)a.c.keys + ((int64_t)pgK * a.c.heads + h) * head +
              (offK + (col & 3)) * d + 8 * grp;
      vp[p] = (const T*)a.c.values + ((int64_t)pgV * a.c.heads + h) * head + col * ps + offV;
      n8[p] = sn - offV;
      all &= n8[p] >= 8;
      any |= n8[p] > 0;
    }
    if (!__any(any)) return;
    all = __all(all);
#pragma unroll
    for (int p = 0; p < kPairs; ++p)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
          kf[2 * p + u][i] = uintx4{};
          if (32 * i + 32 <= sure_values(DP) || 32 * i + 8 * grp < d)
            kf[2 * p + u][i] = *(const uintx4*)(kp[p] + 4 * u * d + 32 * i);
        }
#pragma unroll
    for (int p = 0; p < kPairs; ++p)
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        vf[p][i] = uintx4{};
        if (16 * i + 16 <= sure_values(DP) || 16 * i + col < d) vf[p][i] = *(const uintx4*)(vp[p] + 16 * i * ps);
      }

    floatx4 s[2 * kPairs];
#pragma unroll
    for (int u = 0; u < 2 * kPairs; ++u) {
      s[u] = floatx4{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < kChunks; ++i) s[u] = mfma(__builtin_bit_cast(Tx8, kf[u][i]), q[i], s[u]);
    }
    if (!all) {
      // keys past the token, past the row or of absent pages: whatever their
      // places hold has no weight, NaN and infinities included
#pragma unroll
      for (int p = 0; p < kPairs; ++p) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i >= n8[p]) s[2 * p + i / 4][i % 4] = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < kTiles; ++i) vf[p][i] = keep(vf[p][i], n8[p]);
      }
    }
    Tx8 pr[kPairs];
    weights<kPairs>(s, m, l, c, kBias, o, pr);
#pragma unroll
    for (int p = 0; p < kPairs; ++p)
#pragma unroll
      for (int i = 0; i < kTiles; ++i) o[i] = mfma(__builtin_bit_cast(Tx8, vf[p][i]), pr[p], o[i]);
  }
};

// (m, l) of a row as its logarithm of the sum of exponentials.
__device__ __forceinline__ float lse_of(float m, float l, float scale, float bias) {
  if (m == -__builtin_inff() && l == 0.0f) return m;
  return fmaf(m, scale, kLn2 * (__log2f(l) - bias));
}

// The smallest / largest value of the 16 lanes of a row (lanes 16 g .. 16 g + 15).
template <int CTRL>
__device__ __forceinline__ int row_ror(int x) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_update_dpp(x, x, CTRL, 0xF, 0xF, false);
#else
  return x;
#endif
}
__device__ __forceinline__ int row_min(int x) {
  x = min(x, row_ror<0x128>(x));
  x = min(x, row_ror<0x124>(x));
  x = min(x, row_ror<0x122>(x));
  return min(x, row_ror<0x121>(x));
}
__device__ __forceinline__ int row_max(int x) {
  x = max(x, row_ror<0x128>(x));
  x = max(x, row_ror<0x124>(x));
  x = max(x, row_ror<0x122>(x));
  return max(x, row_ror<0x121>(x));
}

// Tokens of prompts.  A wavefront has as many neighbouring tokens as fill the 16
// columns with their heads of a kv head (two of 8 heads), a workgroup four
// wavefronts.  Neighbours look at much the same blocks: the workgroup walks the
// union of its tokens' blocks, each loaded once, and a wavefront multiplies those
// that a token of its own takes; keys that a column's token does not see get no
// weight.
//
// What bounds it otherwise is loads: a wavefront's MFMA operands straight from
// the cache are 16 bytes of 16 different rows to 16 neighbouring lanes, a row a
// cycle, 64 cycles a load (3,001 tokens of 16 blocks, 4 kv heads of 8, with a
// wavefront for each token: 6.3 GB in 680 us; with four tokens that share one:
// 2.2 GB in 322 us, the same rate).  So tiles of keys and values go to LDS by
// direct loads of neighbouring chunks, a tile ahead of the products, and the
// operands come from there, in chunks that are swapped by row so that 8 lanes
// read from 8 different sets of banks: 246 us.  What bounds it now is the number of
// tiles and the time of each: a workgroup of 8 tokens walks 30 blocks, the union of
// their lists of 16, of which a wavefront uses two thirds; that makes 88 tiles of 64
// keys one after another for each of the 512 workgroups that run at a time, 2.8 us a
// tile, of which products and weights are about 1 us (two wavefronts a SIMD, their
// chain of scores, maxima, exponentials and sums not hidden by one another), the
// rest is waiting for the copy, with one tile ahead, and the barrier.
//
// Without lists every wavefront uses every tile: 4,096 tokens of 8,192 keys (8 kv
// heads of 4, 128 values) 690 us, 600 TFLOP/s.  Operands from LDS, 1 KB and about 10
// cycles each of what four SIMDs share, for an MFMA of 16 cycles, would allow 1,000;
// 6.7 vector instructions an MFMA, in that chain, make the rest.  (32 columns a
// wavefront need more registers than two wavefronts a SIMD have; 192 values over
// lists spill 6 to 10 as it is.)
//
// Lists in any order are right: one that does not ascend is sorted first, and a
// block listed twice counts twice.
//
// A weight of 0 does not hide a value that is not finite.  Values past every
// token's keys are masked; one that only some of the tokens see would reach the
// others' sums as NaN, so a workgroup with a token whose sums are not finite goes
// over its tiles again, where tokens differ in what they see one token after
// another.  An infinity that all see costs 512 tokens of 2,048 keys (64 heads of 64
// values) 126 us, not 54; 4,096 tokens of 8,192 keys 1,839, not 797; over lists of 16
// blocks 1.9 to 5 times as long (16 tokens a wavefront).
constexpr int kSharedWaves = 4;
constexpr int kListInts = 3840;  // of all lists of a workgroup (two workgroups a CU)

// Tokens that share a wavefront, and wavefronts that share a token's heads.
struct Sharing {
  int tokens, tiles;
};
__host__ __device__ __forceinline__ Sharing sharing(int group, int n) {
  if (group > kColumns) return {1, (group + kColumns - 1) / kColumns};
  const int most = kListInts / kSharedWaves / (n + 1);
  const int tokens = kColumns / group;
  return {tokens < most ? tokens : most, 1};
}

// Calls of both kernels (KvAttendArgs::mixed): a span of neighbouring tokens, as many
// as a workgroup of shared wavefronts takes, is a prompt's if one request has its
// first and its last; if the call has at least `least` such spans, their tokens share
// wavefronts and the others do not.  Whether token t (the same for the workgroup's
// 256 threads) is one of them; every kernel of the call finds the same.
__device__ __forceinline__ bool in_prompt(const KvAttendArgs& a, int64_t t) {
  const int64_t spans = a.q.tokens / a.span, mine = t / a.span;
  const auto of_one = [&](int64_t s) {
    const int32_t* r = a.q.token_request + s * a.span;
    return r[0] >= 0 && r[0] == r[a.span - 1];
  };
  if (mine >= spans || !of_one(mine)) return false;
  int64_t found = 0;
  for (int64_t s = 0; s < spans && found < a.least; s += 256)
    found += __syncthreads_count(s + threadIdx.x < spans && of_one(s + threadIdx.x));
  return found >= a.least;
}

// 16 bytes a lane from `from` to lds + 16 lane.
__device__ __forceinline__ void copy16_to_lds(const void* from, void* lds) {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                   (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
#endif
}

// A tile's keys (64 while two workgroups of such tiles fit a CU).
constexpr int tile_keys(int dim) { return dim <= 128 ? 64 : 32; }

// PK: keys of a block in a tile: all of it for pages of 16 and 32, which share a
// tile, else the tile's.
template <int DP, bool BF16, bool LIST, int PK>
struct AttendShared {
  using T = std::conditional_t<BF16, __bf16, _Float16>;
  using Tx8 = std::conditional_t<BF16, bf16x8, halfx8>;
  using Tx4 = std::conditional_t<BF16, bf16x4, halfx4>;
  static constexpr int kKeys = tile_keys(DP);
  static constexpr int kChunks = DP / 32, kTiles = DP / 16;
  // (room for a block that is listed 256 times)
  static constexpr float kBias = BF16 ? 0.0f : 7.0f;
  static constexpr int kNone = kNoBlock;
  // K rows lie at a power of two of 16-byte chunks in LDS, V^T rows densely; 1 KB
  // copies, dealt to the wavefronts
  static constexpr int kRow = DP <= 64 ? 8 : DP <= 128 ? 16 : 32;
  static constexpr int kPerCopy = 1024 * kSharedWaves;
  static constexpr int kCopiesK = kKeys * kRow * 16 / kPerCopy;
  static constexpr int kCopiesV = (kKeys * DP * 2 + kPerCopy - 1) / kPerCopy;
  static constexpr int kBlocks = kKeys / PK;

  // Whole numbers of each of a tile's blocks, 16 bits a block.
  using Counts = std::conditional_t<(kBlocks > 2), uint64_t, uint32_t>;

  // Two buffers with names of their own: loads into one are not taken to alias
  // reads of the other (which would wait for them).
  struct Buffer {
    char *k, *v;
  };
  struct Shared {
    int lists[LIST ? kListInts : 1];
    uint32_t window[kWindow / 32];
    int lowest, again, furthest;
  };

  const KvAttendArgs& a;
  Shared& sh;
  const int lane, wave, col, grp, h;
  const int d, ps;  // values, keys of a page
  const float c;
  Tx8 q[kChunks];
  floatx4 o[kTiles];
  float m, l;
  int pos;       // of the column's token
  int at, next;  // its place in its list, and the block there
  bool on;
  int token, tokens;  // the column's of this wavefront's tokens (-1: none), and their number
  uint32_t from_k[kCopiesK], from_v[kCopiesV];  // what this lane copies, in bytes from a page's
  int block_v;     // ... and whose values
  int at_k, at_v;  // where this lane's first operands are, in bytes

  // Chunks of a row are swapped so that the 8 lanes that read together, rows 0 to
  // 3 and 8 to 11 or neighbours, find 8 sets of banks.
  __device__ __forceinline__ static int swap_of_k(int row) {
    // (alike in both halves of a tile)
    return ((row & 3) | ((row >> 2 ^ row >> 3) & 1) << 2 | (row >> 4 & 1) << 3) & (kRow - 1);
  }
  __device__ __forceinline__ static int swap_of_v(int row) {
    return kKeys == 64 ? row & 7 : (row ^ (row >> 2)) & 3;
  }

  __device__ __forceinline__ AttendShared(const KvAttendArgs& args, Shared& s, int head)
      : a(args), sh(s), lane(threadIdx.x & 63),
        wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)), col(lane & 15), grp(lane >> 4),
        h(head), d(args.c.dim), ps(kBlocks > 1 ? PK : args.c.page), c(args.scale * kLog2e) {
    constexpr int nv = kKeys / 8;
    // (past the head's values: the tile's start, for chunks that nobody uses)
#pragma unroll
    for (int i = 0; i < kCopiesK; ++i) {
      const int x = 64 * (wave + kSharedWaves * i) + lane;
      const int row = x / kRow, chunk = (x % kRow) ^ swap_of_k(row);
      from_k[i] = 8 * chunk < d ? 2 * (row % PK * d + 8 * chunk) : 0;
    }
#pragma unroll
    for (int i = 0; i < kCopiesV; ++i) {
      const int x = 64 * (wave + kSharedWaves * i) + lane;
      const int row = x / nv, chunk = (x % nv) ^ swap_of_v(row);
      from_v[i] = row < d ? 2 * (row * ps + 8 * chunk % PK) : 0;
      block_v = 8 * chunk / PK;  // (the rows of its copies are swapped alike)
    }
    const int r = 8 * (col >> 2) + (col & 3);
    at_k = 16 * (r * kRow + (grp ^ swap_of_k(r)));
    at_v = col * kKeys * 2 + 16 * (grp ^ swap_of_v(col));
  }

  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int i = 0; i < kTiles; ++i) o[i] = floatx4{0, 0, 0, 0};
    m = -__builtin_inff();
    l = 0.0f;
  }

  // The block at the column's place of its list.
  __device__ __forceinline__ int entry() const {
    if (!on) return kNone;
    if constexpr (LIST) return sh.lists[at];
    return at <= pos >> a.c.lps ? at : kNone;
  }

  // How many keys of block b each column sees, and how often it has it listed.
  // Blocks before b that it has listed (their pages are absent) are passed by.
  __device__ __forceinline__ void look(int b, int& seen, int& times) {
    if constexpr (!LIST) {
      seen = on ? min(ps, pos + 1 - (b << a.c.lps)) : 0;
      return;
    }
    times = 0;
    bool some = true;
    while (some) {
      bool moved = false;
      if (next <= b) {
        times += next == b;
        ++at;
        next = entry();
        moved = true;
      }
      some = __any(moved);
    }
    seen = times ? min(ps, pos + 1 - (b << a.c.lps)) : 0;
  }

  // ---- the union of the workgroup's blocks, the same on every wavefront ----------
  uint32_t bits;      // lists: blocks 32 lane .. of the window
  int base, floor;    // the window's first block, the one past its last
  int counter;        // without lists: the next block
  int last;           // the furthest position of the workgroup's tokens

  __device__ __forceinline__ int next_block() {
    if constexpr (!LIST) {
      return counter <= last >> a.c.lps ? counter++ : kNone;
    } else {
      const uint64_t some = __ballot(bits != 0);
      if (!some) return kNone;
      const int i = __builtin_ctzll(some);
      const uint32_t w = __builtin_amdgcn_readlane(bits, i);
      if (lane == i) bits &= bits - 1;
      return base + 32 * i + __builtin_ctz(w);
    }
  }

  struct Tile {
    int block[kBlocks], page[kBlocks], off;
  };
  const int32_t* table;

  // The next tile; false: no more.
  __device__ __forceinline__ bool next_tile(Tile& t) {
    if constexpr (kBlocks == 1) {
      t.off += kKeys;
      if (t.off < ps && t.off < last + 1 - (t.block[0] << a.c.lps)) return true;
    }
    t.off = 0;
    while (true) {
      bool some = false;
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) {
        t.block[i] = block[i];
        t.page[i] = block[i] == kNone || page[i] < 0 || page[i] >= a.c.pages ? -1 : page[i];
        some |= t.page[i] >= 0;
      }
      find();
      if (some) return true;
      if (t.block[kBlocks - 1] == kNone) return false;
    }
  }

  // The blocks after that, looked up a tile ahead.
  int block[kBlocks], page[kBlocks];

  __device__ __forceinline__ void find() {
#pragma unroll
    for (int i = 0; i < kBlocks; ++i) {
      block[i] = next_block();
      page[i] = table_entry(table, block[i] == kNone ? 0 : block[i]);
    }
  }

  // Copies a tile's keys and values into a buffer.
  __device__ __forceinline__ void copy(const Tile& t, Buffer to_) {
    const char *k[kBlocks], *v[kBlocks];
    const int64_t head = (int64_t)ps * d;
#pragma unroll
    for (int i = 0; i < kBlocks; ++i) {
      // (an absent page among others is read as page 0 and not seen)
      const int64_t p = ((int64_t)max(0, t.page[i]) * a.c.heads + h) * head;
      k[i] = (const char*)a.c.keys + 2 * (p + t.off * d);
      v[i] = (const char*)a.c.values + 2 * (p + t.off);
    }
    // (1 KB of keys are rows of one block, often a round of copies is)
    constexpr int kRows = 64 / kRow, kRound = kRows * kSharedWaves;
    const int mine_k = kRound > PK ? kRows * wave / PK : 0;
#pragma unroll
    for (int i = 0; i < kCopiesK; ++i)
      copy16_to_lds(of_block(k, i * kRound / PK + mine_k) + from_k[i],
                    to_.k + 1024 * (wave + kSharedWaves * i));
    const char* mine = of_block(v, block_v);
#pragma unroll
    for (int i = 0; i < kCopiesV; ++i)
      copy16_to_lds(mine + from_v[i], to_.v + 1024 * (wave + kSharedWaves * i));
  }

  // (in registers: a choice among loads would keep the array in memory)
  __device__ __forceinline__ static const char* of_block(const char* const (&x)[kBlocks], int b) {
    const char* y = x[0];
#pragma unroll
    for (int i = 1; i < kBlocks; ++i) {
      const char* z = x[i];
#if defined(__HIP_DEVICE_COMPILE__)
      asm("" : "+s"(z));
#endif
      y = b >= i ? z : y;
    }
    return y;
  }

  // Zeros in the place of values past the workgroup's furthest token, or of an
  // absent page among others: a weight of 0 would not hide what is not finite.
  __device__ __forceinline__ void clear(const Tile& t, Buffer in) {
    constexpr int nv = kKeys / 8, kPer = PK / 8;  // chunks of a row, of a block's
    bool some = false;
    Counts shown = 0;
#pragma unroll
    for (int i = 0; i < kBlocks; ++i) {
      const int n = t.block[i] == kNone || t.page[i] < 0
                        ? 0 : last + 1 - (t.block[i] << a.c.lps) - t.off;
      shown |= (Counts)min(max(0, n), PK) << 16 * i;
      some |= n < PK;
    }
    if (!some) return;
    for (int x = threadIdx.x; x < d * nv; x += 64 * kSharedWaves) {
      const int row = x / nv, chunk = (x % nv) ^ swap_of_v(row);
      const int left = (int)(shown >> 16 * (chunk / kPer) & 0xFFFF) - 8 * (chunk % kPer);
      if (left < 8) *(uintx4*)(in.v + 16 * x) = keep(*(const uintx4*)(in.v + 16 * x), left);
    }
    __syncthreads();
  }

  // 32 keys of a buffer, from key `k0` of the tile on: of this lane's 8 keys its
  // column sees the first n8.  `twice`: log2 of how often a block is listed.
  // EXACT: no value reaches a token that does not see it.
  template <bool EXACT>
  __device__ __forceinline__ void step(Buffer from, int k0, int n8, bool all, float twice) {
    floatx4 s[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      uintx4 kf[kChunks];
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        // (a row 4 further on, and each 4 chunks, differ in one bit of the swap)
        kf[i] = *(const uintx4*)(from.k + 16 * kRow * (k0 + 4 * u) + (at_k ^ (64 * (i ^ u))));
        if (32 * i + 32 > sure_values(DP) && 32 * i + 8 * grp >= d) kf[i] = uintx4{};
      }
      s[u] = floatx4{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < kChunks; ++i)
        s[u] = mfma(__builtin_bit_cast(Tx8, kf[i]), q[i], s[u]);
    }
    // (32 keys on, a chunk's place differs in one bit)
    const char* v = from.v + (at_v ^ (k0 ? 64 : 0));
    uintx4 vf[kTiles];
    if constexpr (!EXACT) {
#pragma unroll
      for (int i = 0; i < kTiles; ++i) vf[i] = *(const uintx4*)(v + i * 32 * kKeys);
    }
    if (!all) hide(s, n8);
    Tx8 pr[1];
    weights<1>(s, m, l, c, kBias + twice, o, pr);
    if constexpr (!EXACT) {
#pragma unroll
      for (int i = 0; i < kTiles; ++i)
        o[i] = mfma(__builtin_bit_cast(Tx8, vf[i]), pr[0], o[i]);
    } else {
      // a token after another, unless all see everything: values that it does not
      // see are zeros to it, and only its columns take the product
#pragma unroll 1
      for (int x = 0; x < tokens; ++x) {
        const int n = all ? 8 : __shfl(n8, 16 * grp + x * a.q.group);
        if (!__any(n > 0)) continue;
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
          const uintx4 vx = keep(*(const uintx4*)(v + i * 32 * kKeys), n);
          const floatx4 y = mfma(__builtin_bit_cast(Tx8, vx), pr[0], o[i]);
          o[i] = all || token == x ? y : o[i];
        }
        if (all) break;
      }
    }
  }

  // A lane's 8 scores of which its column sees the first n.
  __device__ __forceinline__ static void hide(floatx4 (&s)[2], int n) {
    if (__any(n > 0 && n < 8)) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i >= n) s[i / 4][i % 4] = -__builtin_inff();
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i / 4][i % 4] = n > 0 ? s[i / 4][i % 4] : -__builtin_inff();
    }
  }

  // The steps of a tile in a buffer that this wavefront's tokens see; seen and
  // times are kept over the tiles of a block.
  Counts seen, times;

  template <bool EXACT>
  __device__ __forceinline__ void use(const Tile& t, Buffer from) {
    if (t.off == 0) {
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) {
        int n = 0, often = 0;
        if (t.block[i] != kNone) look(t.block[i], n, often);
        if (t.page[i] < 0) n = 0;
        seen = (i ? seen : 0) | (Counts)max(0, n) << 16 * i;
        times = (i ? times : 0) | (Counts)often << 16 * i;
      }
    }
#pragma unroll 1
    for (int k0 = 0; k0 < kKeys; k0 += 32) {
      const int key = k0 + 8 * grp;  // this lane's first
      const int place = 16 * (key / PK % kBlocks);
      const int n8 = (int)(seen >> place & 0xFFFF) - t.off - (kBlocks > 1 ? key % PK : key);
      if (!__any(n8 > 0)) continue;
      const float twice = LIST ? __log2f((float)max(1, (int)(times >> place & 0xFFFF))) : 0.0f;
      step<EXACT>(from, k0, n8, __all(n8 >= 8 || (EXACT && token < 0)), twice);
    }
  }

  uint64_t todo, with;  // tokens of this wavefront: to come, and of the request at hand
  bool open;            // the request at hand may have blocks left

  // Goes to the next request that some wavefront's tokens have; false: none.
  // Every wavefront of the workgroup comes here, and into window().
  __device__ __forceinline__ bool request(int myreq, int stride) {
    __syncthreads();
    if (threadIdx.x == 0) {
      sh.again = kNone;
      sh.furthest = -1;
    }
    __syncthreads();
    int r = todo >> lane & 1 ? myreq : kNone;
#pragma unroll
    for (int x = 32; x >= 1; x >>= 1) r = min(r, __shfl_xor(r, x));
    if (lane == 0 && r != kNone) atomicMin(&sh.again, r);
    __syncthreads();
    r = __builtin_amdgcn_readfirstlane(sh.again);
    if (r == kNone) return false;
    with = todo & __ballot(myreq == r);
    todo &= ~with;
    table = a.q.table + (int64_t)r * a.q.table_stride;
    int far = -1;
    on = token >= 0 && (with >> token & 1);
    at = LIST ? (first_list + max(0, token)) * stride : 0;
    next = entry();
    if (on) far = max(far, pos);
    far = row_max(far);
    if (lane == 0 && far >= 0) atomicMax(&sh.furthest, far);
    __syncthreads();
    last = __builtin_amdgcn_readfirstlane(sh.furthest);
    base = counter = floor = 0;
    return open = true;
  }

  // Makes the union of the request's next blocks, from the lowest that some token
  // has listed on; false: none are left.
  __device__ __forceinline__ bool window(int stride) {
    if constexpr (!LIST) {
      const bool was = open;
      open = false;
      return was;
    }
    // past the last window, whatever of it was absent: every window is a later one
    if (floor > 0) {
      int seen, times;
      look(floor - 1, seen, times);
    }
    __syncthreads();
    if (threadIdx.x < kWindow / 32) sh.window[threadIdx.x] = 0;
    if (threadIdx.x == 0) sh.lowest = kNone;
    __syncthreads();
    int low = next;
    low = row_min(low);
    if (lane == 0 && low != kNone) atomicMin(&sh.lowest, low);
    __syncthreads();
    base = __builtin_amdgcn_readfirstlane(sh.lowest);
    if (base == kNone) return open = false;
    base &= ~(kWindow - 1);
    floor = base + kWindow;
    for (uint64_t left = with; left; left &= left - 1) {
      const int* list = sh.lists + (first_list + __builtin_ctzll(left)) * stride;
      blocks_in_window(list, stride, lane, base, a.q.cols,
                       [&](int b) { atomicOr(&sh.window[b >> 5], 1u << (b & 31)); });
    }
    __syncthreads();
    bits = sh.window[lane];
    return true;
  }

  // All blocks of this wavefront's tokens `todo`.
  template <bool EXACT>
  __device__ __forceinline__ void run(int myreq, int stride, Buffer b0, Buffer b1) {
    Tile now;
    bool more = false;
    open = false;
    const auto turn = [&](Buffer from, Buffer to) {
      Tile then = now;
      more = next_tile(then);
      dma_barrier();  // this tile is there, and the other buffer is free
      mfma_settle();
      if (more) copy(then, to);
      clear(now, from);
      use<EXACT>(now, from);
      now = then;
    };
    // (one loop around the sums, so that they stay in one set of registers)
    while (true) {
      if (!more) {
        while (true) {
          if (!open && !request(myreq, stride)) return;
          if (!window(stride)) continue;
          now.off = 1 << 30;  // (past any block)
          now.block[0] = 0;
          find();
          more = next_tile(now);
          if (more) break;
        }
        __syncthreads();  // (the last tile's buffer is free)
        copy(now, b0);
      }
      turn(b0, b1);
      if (more) turn(b1, b0);
    }
  }

  // The first of the workgroup's lists that is this wavefront's.
  int first_list;
};

template <int DP, bool BF16, bool LIST, int PK>
__global__ __launch_bounds__(64 * kSharedWaves, DP <= 192 ? 2 : 1)
void kv_attend_shared_kernel(KvAttendArgs a) {
  using A = AttendShared<DP, BF16, LIST, PK>;
  __shared__ typename A::Shared sh;
  __shared__ __align__(16) char k0[A::kCopiesK * A::kPerCopy], k1[A::kCopiesK * A::kPerCopy],
      v0[A::kCopiesV * A::kPerCopy], v1[A::kCopiesV * A::kPerCopy];
  const int group = a.q.group;
  const Sharing share = sharing(group, a.n);
  // wavefronts go through the head tiles of a set of tokens, then to the next
  const int h = (int)(blockIdx.x % a.c.heads);
  if (a.mixed && !in_prompt(a, (int64_t)(blockIdx.x / a.c.heads) * a.span)) return;
  A w(a, sh, h);
  const int lane = w.lane;
  const int64_t unit = (int64_t)(blockIdx.x / a.c.heads) * kSharedWaves + w.wave;
  const int mt = (int)(unit % share.tiles);
  const int64_t t0 = unit / share.tiles * share.tokens;
  const int tokens = (int)max<int64_t>(0, min<int64_t>(share.tokens, a.q.tokens - t0));
  // lane i: token t0 + i
  int myreq = -1, mypos = -1;
  if (lane < tokens) {
    myreq = a.q.token_request[t0 + lane];
    mypos = position(a, t0 + lane);
  }
  const bool sees = myreq >= 0 && myreq < a.q.requests && mypos >= 0;
  const int stride = a.n + 1;
  w.first_list = w.wave * share.tokens;
  if constexpr (LIST) {
    // the tokens' lists, without the entries that show nothing, ascending
    for (int i = 0; i < tokens; ++i) {
      const int own = __shfl(sees ? mypos >> a.c.lps : -1, i);
      const int32_t* from = a.blocks + ((t0 + i) * a.c.heads + h) * a.n;
      int* list = sh.lists + (w.first_list + i) * stride;
      int at = 0, before = -1;
      bool ascends = true;
      for (int e = lane; e - lane < a.n; e += 64) {
        const int b = e < a.n ? from[e] : -1;
        const bool take = block_shows(b, a.q.cols, own);
        const uint64_t taken = __ballot(take);
        const uint64_t mine = taken & ((uint64_t(1) << lane) - 1);
        if (take) list[at + (int)__popcll(mine)] = b;
        const int left = __shfl(b, mine ? 63 - __builtin_clzll(mine) : 0);
        ascends &= !take || b >= (mine ? left : before);
        if (taken) before = __shfl(b, 63 - __builtin_clzll(taken));
        at += (int)__popcll(taken);
      }
      end_list(list, at, stride, lane);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if (!__all(ascends)) {
        // each entry's place is the number of those below it, or equal and before
        int b[kKvMaxBlocks / 64], to[kKvMaxBlocks / 64];
#pragma unroll
        for (int x = 0; x < kKvMaxBlocks / 64; ++x) {
          const int e = lane + 64 * x;
          b[x] = e < at ? list[e] : A::kNone;
          to[x] = 0;
          for (int y = 0; y < at; ++y) to[x] += list[y] < b[x] || (list[y] == b[x] && y < e);
        }
#pragma unroll
        for (int x = 0; x < kKvMaxBlocks / 64; ++x)
          if (lane + 64 * x < at) list[to[x]] = b[x];
      }
    }
  }
  const int x = mt * kColumns + w.col;  // column
  const bool mine = x / group < tokens;
  const int tok = mine ? x / group : 0, g = x % group;
  w.pos = __shfl(mypos, tok);
  const auto* src = (const typename A::T*)a.q.q + (t0 + tok) * a.q.q_token +
                    (int64_t)(h * group + g) * a.q.q_head;
#pragma unroll
  for (int i = 0; i < A::kChunks; ++i) {
    uintx4 x4 = {};
    if (mine && 32 * i + 8 * w.grp < a.c.dim) x4 = *(const uintx4*)(src + 32 * i + 8 * w.grp);
    w.q[i] = __builtin_bit_cast(typename A::Tx8, x4);
  }
  const uint64_t seeing = w.todo = __ballot(sees);
  w.token = mine ? tok : -1;
  w.tokens = share.tokens;
  w.reset();
  w.template run<false>(myreq, stride, {k0, v0}, {k1, v1});
  mfma_settle();
  bool good = true;
#pragma unroll
  for (int i = 0; i < A::kTiles; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      good &= fabsf(w.o[i][j]) < __builtin_inff() || 16 * i + 4 * w.grp >= a.c.dim;
  if (__syncthreads_or(!good && mine && (seeing >> tok & 1))) {
    w.todo = seeing;
    w.reset();
    w.template run<true>(myreq, stride, {k0, v0}, {k1, v1});
    mfma_settle();
  }
  const float l = column_sum(w.l);
  if (mine) {
    const float inv = 1.0f / l;
    const int64_t at = ((t0 + tok) * a.c.heads + h) * group + g;
#pragma unroll
    for (int i = 0; i < A::kTiles; ++i) {
      const int d = 16 * i + 4 * w.grp;
      if (d < a.c.dim) {
        typename A::Tx4 x;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          x[j] = (typename A::T)(l == 0.0f ? 0.0f : w.o[i][j] * inv);
        *(typename A::Tx4*)((typename A::T*)a.out + at * a.c.dim + d) = x;
      }
    }
    if (a.lse && w.grp == 0) a.lse[at] = lse_of(w.m, l, a.scale, A::kBias);
  }
}

// A part of a row's keys for each workgroup, its steps dealt to 4 wavefronts in
// turn.  (Eight spare 0.4 us of 12.8 on one token of 777 keys and cost 3 us of
// 45.5 on 256 rows of 2,048.)
template <int DP, bool BF16, bool LIST, bool P16>
__global__ __launch_bounds__(256, 2) void kv_attend_parts_kernel(KvAttendArgs a) {
  constexpr int W = 4;
  using A = Attend<DP, BF16, LIST, P16>;
  __shared__ float so[W][kColumns][DP + 4];
  __shared__ float sm[W][kColumns], sl[W][kColumns];
  const int tiles = (a.q.group + kColumns - 1) / kColumns;
  // first parts first: a row's later ones may be empty, and workgroups go round
  // the 8 XCDs
  const int mt = (int)(blockIdx.x % tiles);
  int64_t b = blockIdx.x / tiles;
  const int h = (int)(b % a.c.heads);
  b /= a.c.heads;
  const int64_t t = b % a.q.tokens;
  const int part = (int)(b / a.q.tokens);
  if (a.mixed && in_prompt(a, t)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  A w(a, threadIdx.x & 63);
  const int r = a.q.token_request[t], pos = position(a, t);
  int64_t k0 = (int64_t)part * a.chunk, k1 = 0;
  int end = 0;
  if (r >= 0 && r < a.q.requests && pos >= 0) {
    end = LIST ? a.n : (pos >> a.c.lps) + 1;
    k1 = (int64_t)end << a.c.lps;
    if (!LIST) k1 = min(k1, (int64_t)pos + 1);
    if (part + 1 < a.splits) k1 = min(k1, k0 + a.chunk);
  }
  w.start(t, h, mt);
  while (k0 < k1) {
    const int e = (int)(k0 >> a.c.lps);
    w.entries(t, h, r, pos, e, end);
    const int64_t stop = min(k1, (int64_t)(e + 64) << a.c.lps);
    for (int64_t k = k0 + wave * A::kKeys; k < stop; k += W * A::kKeys) w.step(h, (int)k);
    k0 = stop;
  }
  w.l = column_sum(w.l);
  const float c = a.scale * kLog2e;
  if (w.grp == 0) {
    sm[wave][w.col] = w.m;
    sl[wave][w.col] = w.l;
  }
#pragma unroll
  for (int i = 0; i < A::kTiles; ++i) *(floatx4*)&so[wave][w.col][16 * i + 4 * w.grp] = w.o[i];
  __syncthreads();
  const int groups = min(kColumns, a.q.group - mt * kColumns);
  const int quads = a.c.dim / 4;
  for (int i = threadIdx.x; i < groups * quads; i += 256) {
    const int g = i / quads, d = 4 * (i % quads);
    float top = sm[0][g];
#pragma unroll
    for (int x = 1; x < W; ++x) top = fmaxf(top, sm[x][g]);
    const float safe = top == -__builtin_inff() ? 0.0f : top;
    float sum = 0.0f;
    floatx4 o = {0, 0, 0, 0};
#pragma unroll
    for (int x = 0; x < W; ++x) {
      const float f = __builtin_amdgcn_exp2f((sm[x][g] - safe) * c);
      sum = fmaf(sl[x][g], f, sum);
      o += *(const floatx4*)&so[x][g][d] * f;
    }
    const int64_t head = t * a.c.heads + h;
    const int gg = mt * kColumns + g;
    if (a.splits == 1) {
      const float inv = 1.0f / sum;
      typename A::Tx4 x;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = (typename A::T)(sum == 0.0f ? 0.0f : o[j] * inv);
      const int64_t at = head * a.q.group + gg;
      *(typename A::Tx4*)((typename A::T*)a.out + at * a.c.dim + d) = x;
      if (a.lse && d == 0) a.lse[at] = lse_of(top, sum, a.scale, A::kBias);
    } else {
      const int64_t at = (head * a.q.group + gg) * a.splits + part;
      *(floatx4*)(a.part_o + at * a.c.dim + d) = o;
      if (d == 0) *(floatx2*)(a.part_ml + 2 * at) = floatx2{top, sum};
    }
  }
}

// Joins the parts of a row: out = sum_s w_s O_s / sum_s w_s l_s, w_s = 2^((m_s -
// max) c).  Threads of one quarter of values take the parts in turn, and their
// sums are added in order: the same result on every run.
template <bool BF16>
__global__ __launch_bounds__(256) void kv_attend_join_kernel(KvAttendArgs a) {
  using T = std::conditional_t<BF16, __bf16, _Float16>;
  using Tx4 = std::conditional_t<BF16, bf16x4, halfx4>;
  __shared__ floatx4 so[256];
  __shared__ float ss[256], sm[4];
  const int tid = threadIdx.x;
  const int64_t at = blockIdx.x;  // (token, query head)
  if (a.mixed && in_prompt(a, at / (a.c.heads * a.q.group))) return;
  const float c = a.scale * kLog2e;
  const float* ml = a.part_ml + 2 * at * a.splits;
  float top = -__builtin_inff();
  for (int s = tid; s < a.splits; s += 256) top = fmaxf(top, ml[2 * s]);
#pragma unroll
  for (int x = 32; x >= 1; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
  if ((tid & 63) == 0) sm[tid >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  const float safe = top == -__builtin_inff() ? 0.0f : top;
  const int quads = a.c.dim / 4, lanes = 256 / quads;
  const int mine = tid / quads, d = 4 * (tid % quads);
  float sum = 0.0f;
  floatx4 o = {0, 0, 0, 0};
  if (mine < lanes) {
    const float* po = a.part_o + at * a.splits * a.c.dim + d;
#pragma unroll 4
    for (int s = mine; s < a.splits; s += lanes) {
      const floatx2 p = *(const floatx2*)(ml + 2 * s);
      const float f = __builtin_amdgcn_exp2f((p[0] - safe) * c);
      sum = fmaf(p[1], f, sum);
      o += *(const floatx4*)(po + (int64_t)s * a.c.dim) * f;
    }
  }
  so[tid] = o;
  ss[tid] = sum;
  __syncthreads();
  if (tid >= quads) return;
  for (int x = 1; x < min(lanes, a.splits); ++x) {
    o += so[x * quads + tid];
    sum += ss[x * quads + tid];
  }
  const float inv = 1.0f / sum;
  Tx4 x;
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = (T)(sum == 0.0f ? 0.0f : o[j] * inv);
  *(Tx4*)((T*)a.out + at * a.c.dim + d) = x;
  if (a.lse && tid == 0) a.lse[at] = lse_of(top, sum, a.scale, kBiasOf<T>);
}

int64_t shared_grid(const KvAttendArgs& a) {
  const Sharing sh = sharing(a.q.group, a.n);
  const int64_t units = (a.q.tokens + sh.tokens - 1) / sh.tokens * sh.tiles;
  return (units + kSharedWaves - 1) / kSharedWaves * a.c.heads;
}

template <int DP, bool BF16, bool LIST, bool P16>
void launch_parts(const KvAttendArgs& a, hipStream_t s) {
  const int tiles = (a.q.group + kColumns - 1) / kColumns;
  const dim3 grid((unsigned)(a.q.tokens * a.c.heads * tiles * a.splits));
  kv_attend_parts_kernel<DP, BF16, LIST, P16><<<grid, 256, 0, s>>>(a);
}

template <int DP, bool BF16, bool LIST>
void launch_listed(const KvAttendArgs& a, hipStream_t s) {
  if (!a.shared) {
    if (a.c.page == 16) launch_parts<DP, BF16, LIST, true>(a, s);
    else launch_parts<DP, BF16, LIST, false>(a, s);
  }
  if (!a.shared && !a.mixed) return;
  const dim3 grid((unsigned)shared_grid(a));
  constexpr int kThreads = 64 * kSharedWaves;
  constexpr int kKeys = tile_keys(DP);
  if (a.c.page == 16)
    kv_attend_shared_kernel<DP, BF16, LIST, 16><<<grid, kThreads, 0, s>>>(a);
  else if (kKeys > 32 && a.c.page == 32)
    kv_attend_shared_kernel<DP, BF16, LIST, 32><<<grid, kThreads, 0, s>>>(a);
  else
    kv_attend_shared_kernel<DP, BF16, LIST, kKeys><<<grid, kThreads, 0, s>>>(a);
}

template <int DP, bool BF16>
void launch_dim(const KvAttendArgs& a, hipStream_t s) {
  a.blocks ? launch_listed<DP, BF16, true>(a, s) : launch_listed<DP, BF16, false>(a, s);
}

template <bool BF16>
void launch_type(const KvAttendArgs& a, hipStream_t s) {
  if (a.c.dim <= 64) launch_dim<64, BF16>(a, s);
  else if (a.c.dim <= 96) launch_dim<96, BF16>(a, s);
  else if (a.c.dim <= 128) launch_dim<128, BF16>(a, s);
  else if (a.c.dim <= 192) launch_dim<192, BF16>(a, s);
  else launch_dim<256, BF16>(a, s);
}

// Whether tokens of prompts share wavefronts.  A row by itself reads its keys,
// 57 ns for 1,024 of them with the card full; a workgroup of shared wavefronts
// walks its requests' keys or the union of their lists, about 25 and 12 us for
// 1,024, and 384 workgroups run at a time.  Measured (16 bits, 128 values, 8 kv
// heads of 4), a row by itself / shared:
//   4,096 keys: one request of 32 tokens 64 / 96 us, of 64 122 / 96, of 512 873 /
//   100; up to 2,048 keys: 32 requests of 4 tokens 105 / 170, of 8 184 / 94;
//   64 requests of 4 176 / 153;
//   lists of 16 of 256 blocks of 64: one request of 128 tokens 62 / 73, of 256
//   118 / 75, of 512 230 / 77; 64 requests of 4 130 / 218 (131 / 123 with 8 heads a
//   kv head), 128 requests of 4 252 / 236; 128 of 2 149 / 189 (8 heads);
//   lists of 64 of 1,024 blocks of 16: one request of 256 81 / 101;
//   256 values, 4,096 keys: one request of 64 tokens 234 / 198, of 128 456 / 202.
//
// The cost of a workgroup's walk for `tokens` tokens, `each` to a request, in those
// figures' measure.
int64_t cost_of_walk(const KvAttendArgs& a, int64_t tokens, int64_t each) {
  int64_t walks = 1 + (tokens - 1) / each;  // requests, each its keys or the union of
  if (a.n) {                                // some lists, which overlap
    const int64_t lists = std::min(tokens, each), apart = std::max(1, a.q.cols / a.n);
    walks *= std::max<int64_t>(1, lists * apart / (lists + apart));
    if (a.c.page == 16) walks *= 2;
  }
  return (a.n ? 220 : 480) * walks;
}

bool shares(const KvAttendArgs& a, int64_t rows) {
  const int64_t each = a.q.tokens / std::max<int64_t>(1, a.q.requests);
  if (each < 3) return false;
  const Sharing sh = sharing(a.q.group, a.n);
  const int64_t tokens = std::max(1, sh.tokens * kSharedWaves / sh.tiles);  // of a workgroup
  return rows * 384 >= cost_of_walk(a, tokens, each) * std::max<int64_t>(384, shared_grid(a));
}

// Whether both kernels run: a call of fewer than three tokens a row of the table may
// still hold a prompt, the other rows being idle or having a token each, which the
// device finds (in_prompt).  One kernel / both, 4,096 keys, 256 rows (8 kv heads of 4,
// 128 values): one row with 512 tokens, the others idle 874 / 162 us (3,523 / 425 over
// 16,384 keys), with a token each 1,551 / 856, 128 tokens so 913 / 825, 16 706 / 713;
// no prompt 690 / 697 and 330 / 331 for 128 rows, which is what the second launch and
// the workgroups that find nothing cost.  So it is made where rows by themselves
// take 0.45 ms; lists: 512 tokens and 500 single ones of 32 blocks 1,118 / 802, none
// and 1,024 of 16 695 / 696.
void mix(KvAttendArgs& a, int64_t rows, int64_t most) {
  const Sharing sh = sharing(a.q.group, a.n);
  if (sh.tiles > 1 || rows * most < 8 << 20) return;
  a.span = sh.tokens * kSharedWaves;
  const int64_t cost = cost_of_walk(a, a.span, a.span), per = (int64_t)a.span * a.c.heads;
  a.least = (int)((cost + per - 1) / per);
  a.mixed = a.span * 384 >= cost && a.q.tokens / a.span >= a.least;
}

}  // namespace

void kv_attend_plan(KvAttendArgs& a) {
  const int tiles = (a.q.group + kColumns - 1) / kColumns;
  const int64_t rows = a.q.tokens * a.c.heads * tiles;
  const int64_t most = a.n ? (int64_t)a.n << a.c.lps
                                : std::min<int64_t>(a.longest, (int64_t)a.q.cols << a.c.lps);
  a.splits = 1;
  a.chunk = 64;
  a.shared = a.mixed = false;
  if (rows == 0) return;
  if (shares(a, rows)) {
    a.shared = true;
    return;
  }
  // As many parts as fill the card (2 workgroups a CU: chunks of 4,096 instead
  // of 1,024 keys 187 / 199 us on one request of 262,144 tokens and 8 kv heads),
  // but no longer ones than 1,024 keys where requests differ in length (64
  // ragged requests of up to 8,192 tokens, 8 kv heads: 247 us with 1,024, 260
  // with 4,096).  Rows of up to 1,024 keys stay whole: the launch that joins
  // parts costs more than the wait (777 keys, 8 heads: 13.1 us whole, 15.3 in
  // four), and so do lists where there is a row for every CU (256 rows of 2,048
  // keys: 51.5 us whole, 55.4 in two).
  const bool whole = most <= 1024 || (a.n && rows >= 256);
  int64_t chunk = (most * rows / 512 + 255) / 256 * 256;
  if (a.q.tokens > 1 && !a.n) {
    // nor more than 16,384 parts over all rows: a table may be far wider than its
    // requests are long, and a part costs a workgroup and its place in the
    // workspace.  Without a limit / with it (8 kv heads of 4, 128 values): 1,024
    // requests of up to 8,192 tokens 3,359 / 3,073 us, and 4,118 / 2,954 in a table
    // for 32,768; 256 of up to 2,048 in a table for 131,072 1,203 / 268; 4,096 of up
    // to 1,500 in one for 4,096 2,889 / 2,219.  (65,536 parts: 3,370, 3,127, 447,
    // 2,606; 8,192: 2,989, 2,889, 241, 2,216, but 300, not 266, for 64 of up to 8,192
    // in a table for 131,072.)
    const int64_t least = (most * rows / 16384 + 255) / 256 * 256;
    chunk = std::max(least, std::min<int64_t>(chunk, 1024));
  } else if (!a.n && a.longest == INT32_MAX) {
    // A single token whose history nobody tells: most of the table may be empty, so
    // parts of 2,048 keys, unless that makes more than 2,048 parts.  Without / with
    // it (8 kv heads of 4, 128 values), in a table for 1,048,576 tokens: 777 keys
    // 20.7 / 24.5 us, 16,000 224 / 67, 131,072 256 / 96, all 627 / 644; for 262,144:
    // 777 keys 20.9 / 22.0, 16,000 64.5 / 38.1, 131,072 98.6 / 104, all 189 / 191.
    chunk = std::min(chunk, std::max<int64_t>(2048, most * rows / 2048));
  }
  chunk = std::max<int64_t>(512, std::min<int64_t>(chunk, 1 << 30));
  if (!whole) a.splits = (int)((most + chunk - 1) / chunk);
  a.chunk = whole ? 1 << 30 : (int)chunk;
  mix(a, rows, most);
}

int64_t kv_attend_workspace(const KvAttendArgs& a) {
  if (a.splits <= 1) return 0;
  return a.q.tokens * a.c.heads * a.q.group * a.splits * (a.c.dim + 2) * 4;
}

int64_t kv_attend_grid(const KvAttendArgs& a) {
  if (a.shared) return shared_grid(a);
  const int64_t rows = a.q.tokens * a.c.heads * ((a.q.group + kColumns - 1) / kColumns);
  const int64_t join = a.splits > 1 ? a.q.tokens * a.c.heads * a.q.group : 0;
  return std::max({rows * a.splits, join, a.mixed ? shared_grid(a) : 0});
}

hipError_t launch_kv_attend(const KvAttendArgs& a, hipStream_t s) {
  a.c.bf16 ? launch_type<true>(a, s) : launch_type<false>(a, s);
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  if (a.splits > 1) {
    const unsigned grid = (unsigned)(a.q.tokens * a.c.heads * a.q.group);
    if (a.c.bf16) kv_attend_join_kernel<true><<<grid, 256, 0, s>>>(a);
    else kv_attend_join_kernel<false><<<grid, 256, 0, s>>>(a);
  }
  return hipGetLastError();
}

}  // namespace mlxvs::kern
