// Attention of new tokens over the paged key-value cache: over every block up
// to the token's position, or over the blocks of a list of its own.
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - max)
//
// over the keys j that the token sees, one pass with the running maximum and
// sum.  The G query heads of a kv head are the 16 columns of the products:
// S^T = K Q^T and O^T = V^T P^T, both on the 16x16x32 MFMA (bf16 / f16 in,
// float32 out).  With values transposed within a page, K rows and V^T rows are
// 16-byte loads in the A operand's own layout, so nothing goes through LDS; and
// S^T comes out with its keys along the registers.  The keys of a 32-key pair
// of S tiles are dealt to the tiles' rows so that a lane ends up with 8
// consecutive keys (row m of tile t is key 8 (m / 4) + 4 t + m % 4): exactly
// the 8 keys it holds of the second product's B operand, so P stays in its
// registers too, and the V^T loads stay 16 bytes wide.
//
// P is rounded to the cache's type for the second product (the values' own
// precision; a sum of roundings that averages out), its sum is not; under f16
// P is scaled by 2^14 so that small terms of long sums stay normal numbers.
// Scores, maxima, sums and the output are float32.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "kv_cache.h"

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
  static constexpr float kBias = BF16 ? 0.0f : 14.0f;  // log2 of P's scale

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
    float top = m;
#pragma unroll
    for (int u = 0; u < 2 * kPairs; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, s[u][i]);
    top = column_max(top);
    if (__any(top > m)) {
      // (a column that has seen nothing: 2^(-inf))
      const float w = top == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f((m - top) * c);
      l *= w;
#pragma unroll
      for (int i = 0; i < kTiles; ++i) o[i] *= w;
      m = top;
    }
    const float base = kBias - (m == -__builtin_inff() ? 0.0f : m) * c;
    Tx8 pr[kPairs];
#pragma unroll
    for (int p = 0; p < kPairs; ++p)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = __builtin_amdgcn_exp2f(fmaf(s[2 * p + i / 4][i % 4], c, base));
        l += x;
        pr[p][i] = (T)x;
      }
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

// Tokens of prompts: a wavefront for as many neighbouring tokens as fill NT
// tiles of 16 columns with their heads of a kv head (two tokens of 8 heads in a
// tile).  Neighbours look at much the same blocks: their lists are merged block
// by block, always the lowest of the tokens' next ones, so that a block that
// several of them take is loaded once and multiplied by all their heads, and
// keys that a column's token does not see get no weight.  What bounds it is
// loads from L2 and the Infinity Cache: with a wavefront for each token 3,001
// tokens of 16 blocks, 4 kv heads of 8, read 6.3 GB in 680 us.
//
// Lists in any order are right: each entry is taken once, whatever it meets.
//
// A weight of 0 does not hide a value that is not finite.  Values past every
// token's keys are masked; one that only some of the tokens see would reach the
// others' sums as NaN, so a wavefront whose sums are not finite does its tokens
// over, one at a time.
extern __shared__ int kv_lists[];  // [tokens][n + 1]

template <int DP, bool BF16, bool LIST, bool P16, int NT>
struct AttendShared {
  using T = std::conditional_t<BF16, __bf16, _Float16>;
  using Tx8 = std::conditional_t<BF16, bf16x8, halfx8>;
  using Tx4 = std::conditional_t<BF16, bf16x4, halfx4>;
  static constexpr int kChunks = DP / 32, kTiles = DP / 16;
  static constexpr float kBias = BF16 ? 0.0f : 14.0f;
  static constexpr int kNone = 0x7FFFFFFF;

  const KvAttendArgs& a;
  const int lane, col, grp, h;
  const float c;
  Tx8 q[NT][kChunks];
  floatx4 o[NT][kTiles];
  float m[NT], l[NT];
  int pos[NT];               // of the column's token
  // the column's place in its token's list (in LDS; without lists, counting
  // up) and its next block
  int at[NT], next[NT];
  bool on[NT];

  __device__ __forceinline__ AttendShared(const KvAttendArgs& args, int ln, int head)
      : a(args), lane(ln), col(ln & 15), grp(ln >> 4), h(head), c(args.scale * kLog2e) {}

  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < kTiles; ++i) o[n][i] = floatx4{0, 0, 0, 0};
      m[n] = -__builtin_inff();
      l[n] = 0.0f;
    }
  }

  __device__ __forceinline__ int entry(int n) const {
    if (!on[n]) return kNone;
    if constexpr (LIST) return kv_lists[at[n]];
    return at[n] <= min(pos[n] >> a.c.lps, a.q.cols - 1) ? at[n] : kNone;
  }

  // The lowest next block of the columns that are on (kNone: no more), and how
  // many of its keys each column sees.
  __device__ __forceinline__ int advance(int (&seen)[NT]) {
    int b = next[0];
#pragma unroll
    for (int n = 1; n < NT; ++n) b = min(b, next[n]);
    b = __builtin_amdgcn_readfirstlane(row_min(b));
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const bool hit = next[n] == b && b != kNone;
      seen[n] = hit ? min(a.c.page, pos[n] + 1 - (b << a.c.lps)) : 0;
      if (hit) {
        ++at[n];
        next[n] = entry(n);
      }
    }
    return b;
  }

  // What one look at the lists gives: the keys of a block (of two pages of 16).
  struct Unit {
    const T *k, *v;  // this lane's K row and V^T row of its first 32 keys
    int lim[NT];     // of those, and this lane's 8, the first that a column sees
    int top;         // keys that any column sees
    bool all;        // every column sees all
  };
  // blocks looked up ahead, so that their pages are known in time
  static constexpr int kBlocks = P16 ? 2 : 1;
  int block[kBlocks], page[kBlocks], seen[kBlocks][NT];

  __device__ __forceinline__ void look(const int32_t* table) {
#pragma unroll
    for (int i = 0; i < kBlocks; ++i) {
      block[i] = advance(seen[i]);
      page[i] = table_entry(table, block[i] == kNone ? 0 : block[i]);
    }
  }

  // The next unit whose pages are there; false: no more.
  __device__ __forceinline__ bool unit(const int32_t* table, Unit& u) {
    const int ps = P16 ? 16 : a.c.page, d = a.c.dim;
    const int64_t head = (int64_t)ps * d;
    while (block[0] != kNone) {
      bool there[kBlocks], some = false;
      int p[kBlocks];
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) {
        there[i] = block[i] != kNone && page[i] >= 0 && page[i] < a.c.pages;
        some |= there[i];
        p[i] = there[i] ? page[i] : 0;  // (an absent page is read as page 0 and not seen)
      }
      if (some) {
        const int row = 8 * (col >> 2);  // this lane's K rows start here
        int64_t pk = p[0], pv = p[0];
        if constexpr (P16) {
          pk = row < 16 ? p[0] : p[1];
          pv = grp < 2 ? p[0] : p[1];
        }
        u.k = (const T*)a.c.keys + (pk * a.c.heads + h) * head +
              ((P16 ? row & 15 : row) + (col & 3)) * d + 8 * grp;
        u.v = (const T*)a.c.values + (pv * a.c.heads + h) * head + col * ps +
              (P16 ? (8 * grp) & 15 : 8 * grp);
        int top = 0;
        u.all = true;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          int s = there[0] ? seen[0][n] : 0;
          if constexpr (P16) {
            const int s1 = there[1] ? seen[1][n] : 0;
            top = max(top, s1 > 0 ? 16 + s1 : s);
            u.all &= s == 16 && s1 == 16;
            u.lim[n] = (grp < 2 ? s : s1) - ((8 * grp) & 15);
          } else {
            top = max(top, s);
            u.all &= s == ps;
            u.lim[n] = s - 8 * grp;
          }
        }
        u.top = __builtin_amdgcn_readfirstlane(row_max(top));
        u.all = __all(u.all);
      }
      look(table);
      if (some) return true;
    }
    return false;
  }

  // Loads without conditions, so that the waits count them: values past the
  // head's are read in a place of its own and masked (K), or make sums that
  // nobody stores (V).
  __device__ __forceinline__ void load_k(uintx4 (&kf)[2][kChunks], const T* kp) const {
    const int d = a.c.dim;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        int at = 32 * i;
        if (32 * i + 32 > sure_values(DP) && 32 * i + 8 * grp >= d) at = -8 * grp;
        kf[u][i] = *(const uintx4*)(kp + 4 * u * d + at);
      }
  }
  __device__ __forceinline__ Tx8 k_row(const uintx4 (&kf)[kChunks], int i) const {
    uintx4 x = kf[i];
    if (32 * i + 32 > sure_values(DP) && 32 * i + 8 * grp >= a.c.dim) x = uintx4{};
    return __builtin_bit_cast(Tx8, x);
  }
  __device__ __forceinline__ void load_v(uintx4 (&vf)[kTiles], const T* vp) const {
    const int d = a.c.dim, ps = P16 ? 16 : a.c.page;
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      int row = 16 * i;
      if (16 * i + 16 > sure_values(DP) && 16 * i + col >= d) row = -col;
      vf[i] = *(const uintx4*)(vp + row * ps);
    }
  }

  // All blocks of the columns that are on, of request r, 32 keys a step; the K
  // rows of the next step are on their way while this one's weights are made.
  __device__ __forceinline__ void run(int r) {
    const int d = a.c.dim;
    const int32_t* table = a.q.table + (int64_t)r * a.q.table_stride;
#pragma unroll
    for (int n = 0; n < NT; ++n) next[n] = entry(n);
    look(table);
    Unit u;
    if (!unit(table, u)) return;
    uintx4 kf[2][kChunks], vf[kTiles];
    load_k(kf, u.k);
    int off = 0;
    for (bool more = true; more;) {
      load_v(vf, u.v + off);
      floatx4 s[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          s[n][x] = floatx4{0, 0, 0, 0};
#pragma unroll
          for (int i = 0; i < kChunks; ++i)
            s[n][x] = mfma(k_row(kf[x], i), q[n][i], s[n][x]);
        }
      // this step's limits, then the next step
      int n8[NT], most = 0;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        n8[n] = u.lim[n] - off;
        most = max(most, n8[n]);
      }
      const bool all = u.all;
      off += 32;
      if (off >= u.top) {
        off = 0;
        more = unit(table, u);
      }
      load_k(kf, u.k + off * d);  // (after the last step: its own once more)
      Tx8 pr[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if (!all) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (i >= n8[n]) s[n][i / 4][i % 4] = -__builtin_inff();
        }
        float top = m[n];
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, s[n][i / 4][i % 4]);
        top = column_max(top);
        if (__any(top > m[n])) {
          const float w = top == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f((m[n] - top) * c);
          l[n] *= w;
#pragma unroll
          for (int i = 0; i < kTiles; ++i) o[n][i] *= w;
          m[n] = top;
        }
        const float base = kBias - (m[n] == -__builtin_inff() ? 0.0f : m[n]) * c;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float x = __builtin_amdgcn_exp2f(fmaf(s[n][i / 4][i % 4], c, base));
          l[n] += x;
          pr[n][i] = (T)x;
        }
      }
      if (!all) {
        most = row_max(most);
        if (__any(most < 8)) {
#pragma unroll
          for (int i = 0; i < kTiles; ++i) vf[i] = keep(vf[i], most);
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < kTiles; ++i)
          o[n][i] = mfma(__builtin_bit_cast(Tx8, vf[i]), pr[n], o[n][i]);
    }
  }
};

template <int DP>
constexpr int kColumnTiles = DP <= 128 ? 2 : 1;  // (registers: two wavefronts a SIMD)

// Tokens that share a wavefront, and wavefronts that share a token's heads.
struct Sharing {
  int tokens, tiles;
};
__host__ __device__ __forceinline__ Sharing sharing(int group, int columns) {
  if (group <= columns) return {columns / group, 1};
  return {1, (group + columns - 1) / columns};
}

template <int DP, bool BF16, bool LIST, bool P16>
__global__ __launch_bounds__(64, 2) void kv_attend_shared_kernel(KvAttendArgs a) {
  constexpr int NT = kColumnTiles<DP>;
  using A = AttendShared<DP, BF16, LIST, P16, NT>;
  const int group = a.q.group, lane = threadIdx.x;
  const Sharing sh = sharing(group, kColumns * NT);
  const int mt = (int)(blockIdx.x % sh.tiles);
  const int h = (int)(blockIdx.x / sh.tiles % a.c.heads);
  const int64_t t0 = (int64_t)(blockIdx.x / sh.tiles / a.c.heads) * sh.tokens;
  const int tokens = (int)min<int64_t>(sh.tokens, a.q.tokens - t0);
  A w(a, lane, h);
  // lane i: token t0 + i
  int myreq = -1, mypos = -1;
  if (lane < tokens) {
    myreq = a.q.token_request[t0 + lane];
    mypos = a.q.positions[t0 + lane];
  }
  const bool sees = myreq >= 0 && myreq < a.q.requests && mypos >= 0;
  if constexpr (LIST) {
    // the tokens' lists, without the entries that show nothing
    for (int i = 0; i < tokens; ++i) {
      const int own = __shfl(sees ? mypos >> a.c.lps : -1, i);
      const int32_t* from = a.blocks + ((t0 + i) * a.c.heads + h) * a.n;
      int at = i * (a.n + 1);
      for (int e = lane; e - lane < a.n; e += 64) {
        const int b = e < a.n ? from[e] : -1;
        const bool take = b >= 0 && b < a.q.cols && b <= own;
        const uint64_t taken = __ballot(take);
        if (take) kv_lists[at + (int)__popcll(taken & ((uint64_t(1) << lane) - 1))] = b;
        at += (int)__popcll(taken);
      }
      if (lane == 0) kv_lists[at] = A::kNone;
    }
    __syncthreads();
  }
  int tok[NT], g[NT];
  bool mine[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int x = mt * kColumns * NT + kColumns * n + w.col;  // column
    tok[n] = x / group;
    g[n] = x % group;
    mine[n] = tok[n] < tokens;
    if (!mine[n]) tok[n] = 0;
    w.pos[n] = __shfl(mypos, tok[n]);
    const auto* src = (const typename A::T*)a.q.q + (t0 + tok[n]) * a.q.q_token +
                      (int64_t)(h * group + g[n]) * a.q.q_head;
#pragma unroll
    for (int i = 0; i < A::kChunks; ++i) {
      uintx4 x4 = {};
      if (mine[n] && 32 * i + 8 * w.grp < a.c.dim) x4 = *(const uintx4*)(src + 32 * i + 8 * w.grp);
      w.q[n][i] = __builtin_bit_cast(typename A::Tx8, x4);
    }
  }
  // first all tokens together, a request after another; then, if that left
  // sums that are not finite, each token by itself
  for (int alone = -1; alone < tokens; ++alone) {
    w.reset();
    uint64_t todo = __ballot(sees);
    if (alone >= 0) todo &= uint64_t(1) << alone;
    while (todo) {
      const int r = __builtin_amdgcn_readlane(myreq, __builtin_ctzll(todo));
      const uint64_t with = todo & __ballot(myreq == r);
      todo &= ~with;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        w.on[n] = mine[n] && (with >> tok[n] & 1);
        w.at[n] = LIST ? tok[n] * (a.n + 1) : 0;
      }
      w.run(r);
    }
    bool good = true;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < A::kTiles; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          good &= fabsf(w.o[n][i][j]) < __builtin_inff() || 16 * i + 4 * w.grp >= a.c.dim;
    if (alone < 0 && !__all(good) && tokens > 1) continue;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float l = column_sum(w.l[n]);
      if (!mine[n] || (alone >= 0 && tok[n] != alone)) continue;
      const float inv = 1.0f / l;
      const int64_t at = ((t0 + tok[n]) * a.c.heads + h) * group + g[n];
#pragma unroll
      for (int i = 0; i < A::kTiles; ++i) {
        const int d = 16 * i + 4 * w.grp;
        if (d < a.c.dim) {
          typename A::Tx4 x;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            x[j] = (typename A::T)(l == 0.0f ? 0.0f : w.o[n][i][j] * inv);
          *(typename A::Tx4*)((typename A::T*)a.out + at * a.c.dim + d) = x;
        }
      }
      if (a.lse && w.grp == 0) a.lse[at] = lse_of(w.m[n], l, a.scale, A::kBias);
    }
    if (alone < 0) break;
  }
}

// A part of a row's keys for each workgroup, its steps dealt to the W wavefronts
// in turn.
template <int DP, bool BF16, bool LIST, bool P16, int W>
__global__ __launch_bounds__(64 * W, 2) void kv_attend_parts_kernel(KvAttendArgs a) {
  constexpr int H = 4;  // wavefronts whose sums meet in LDS at a time
  using A = Attend<DP, BF16, LIST, P16>;
  __shared__ float so[H][kColumns][DP + 4];
  __shared__ float sm[H][kColumns], sl[H][kColumns];
  const int tiles = (a.q.group + kColumns - 1) / kColumns;
  // first parts first: a row's later ones may be empty, and workgroups go round
  // the 8 XCDs
  const int mt = (int)(blockIdx.x % tiles);
  int64_t b = blockIdx.x / tiles;
  const int h = (int)(b % a.c.heads);
  b /= a.c.heads;
  const int64_t t = b % a.q.tokens;
  const int part = (int)(b / a.q.tokens);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  A w(a, threadIdx.x & 63);
  const int r = a.q.token_request[t], pos = a.q.positions[t];
  int64_t k0 = (int64_t)part * a.chunk, k1 = 0;
  int end = 0;
  if (r >= 0 && r < a.q.requests && pos >= 0) {
    end = LIST ? a.n : min(pos >> a.c.lps, a.q.cols - 1) + 1;
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
  const auto put = [&](int x) {
    if (w.grp == 0) {
      sm[x][w.col] = w.m;
      sl[x][w.col] = w.l;
    }
#pragma unroll
    for (int i = 0; i < A::kTiles; ++i) *(floatx4*)&so[x][w.col][16 * i + 4 * w.grp] = w.o[i];
  };
  if constexpr (W > H) {
    static_assert(W == 2 * H, "pairs of wavefronts");
    if (wave >= H) put(wave - H);
    __syncthreads();
    if (wave < H) {
      const float m = sm[wave][w.col], top = fmaxf(w.m, m);
      const float safe = top == -__builtin_inff() ? 0.0f : top;
      const float f0 = __builtin_amdgcn_exp2f((w.m - safe) * c);
      const float f1 = __builtin_amdgcn_exp2f((m - safe) * c);
      w.m = top;
      w.l = w.l * f0 + sl[wave][w.col] * f1;
#pragma unroll
      for (int i = 0; i < A::kTiles; ++i)
        w.o[i] = w.o[i] * f0 + *(const floatx4*)&so[wave][w.col][16 * i + 4 * w.grp] * f1;
      put(wave);  // (in the places that this lane has read)
    }
  } else {
    put(wave);
  }
  __syncthreads();
  const int groups = min(kColumns, a.q.group - mt * kColumns);
  const int quads = a.c.dim / 4;
  for (int i = threadIdx.x; i < groups * quads; i += 64 * W) {
    const int g = i / quads, d = 4 * (i % quads);
    float top = sm[0][g];
#pragma unroll
    for (int x = 1; x < H; ++x) top = fmaxf(top, sm[x][g]);
    const float safe = top == -__builtin_inff() ? 0.0f : top;
    float sum = 0.0f;
    floatx4 o = {0, 0, 0, 0};
#pragma unroll
    for (int x = 0; x < H; ++x) {
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
  if (a.lse && tid == 0) a.lse[at] = lse_of(top, sum, a.scale, BF16 ? 0.0f : 14.0f);
}

int column_tiles(int dim) { return dim <= 128 ? kColumnTiles<128> : kColumnTiles<256>; }

int64_t shared_grid(const KvAttendArgs& a) {
  const Sharing sh = sharing(a.q.group, kColumns * column_tiles(a.c.dim));
  return (a.q.tokens + sh.tokens - 1) / sh.tokens * a.c.heads * sh.tiles;
}

template <int DP, bool BF16, bool LIST, bool P16>
void launch_one(const KvAttendArgs& a, hipStream_t s) {
  if (a.waves == 1) {
    const Sharing sh = sharing(a.q.group, kColumns * kColumnTiles<DP>);
    const size_t lds = LIST ? sizeof(int) * sh.tokens * (a.n + 1) : 0;
    kv_attend_shared_kernel<DP, BF16, LIST, P16>
        <<<dim3((unsigned)shared_grid(a)), 64, lds, s>>>(a);
    return;
  }
  const int tiles = (a.q.group + kColumns - 1) / kColumns;
  const dim3 grid((unsigned)(a.q.tokens * a.c.heads * tiles * a.splits));
  if (a.waves == 8) kv_attend_parts_kernel<DP, BF16, LIST, P16, 8><<<grid, 512, 0, s>>>(a);
  else kv_attend_parts_kernel<DP, BF16, LIST, P16, 4><<<grid, 256, 0, s>>>(a);
}

template <int DP, bool BF16>
void launch_dim(const KvAttendArgs& a, hipStream_t s) {
  const bool p16 = a.c.page == 16;
  if (a.blocks) {
    p16 ? launch_one<DP, BF16, true, true>(a, s) : launch_one<DP, BF16, true, false>(a, s);
  } else {
    p16 ? launch_one<DP, BF16, false, true>(a, s) : launch_one<DP, BF16, false, false>(a, s);
  }
}

template <bool BF16>
void launch_type(const KvAttendArgs& a, hipStream_t s) {
  if (a.c.dim <= 64) launch_dim<64, BF16>(a, s);
  else if (a.c.dim <= 96) launch_dim<96, BF16>(a, s);
  else if (a.c.dim <= 128) launch_dim<128, BF16>(a, s);
  else if (a.c.dim <= 192) launch_dim<192, BF16>(a, s);
  else launch_dim<256, BF16>(a, s);
}

}  // namespace

void kv_attend_plan(KvAttendArgs& a) {
  const int tiles = (a.q.group + kColumns - 1) / kColumns;
  const int64_t rows = a.q.tokens * a.c.heads * tiles;
  const int64_t most = a.n ? (int64_t)a.n << a.c.lps
                                : std::min<int64_t>(a.longest, (int64_t)a.q.cols << a.c.lps);
  a.splits = 1;
  a.chunk = 64;
  a.waves = 4;
  if (rows == 0) return;
  // tokens of prompts share wavefronts, if that leaves enough of them
  if (a.q.tokens >= 4 * a.q.requests && shared_grid(a) >= 1024) {
    a.waves = 1;
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
  if (a.q.tokens > 1 && !a.n) chunk = std::min<int64_t>(chunk, 1024);
  chunk = std::max<int64_t>(512, std::min<int64_t>(chunk, 1 << 30));
  if (!whole) a.splits = (int)((most + chunk - 1) / chunk);
  a.chunk = whole ? 1 << 30 : (int)chunk;
  // eight wavefronts share a part where there is no second workgroup for a CU
  if (rows * a.splits <= 256) a.waves = 8;
}

int64_t kv_attend_workspace(const KvAttendArgs& a) {
  if (a.splits <= 1) return 0;
  return a.q.tokens * a.c.heads * a.q.group * a.splits * (a.c.dim + 2) * 4;
}

int64_t kv_attend_grid(const KvAttendArgs& a) {
  if (a.waves == 1) return shared_grid(a);
  const int64_t rows = a.q.tokens * a.c.heads * ((a.q.group + kColumns - 1) / kColumns);
  return std::max(a.q.tokens * a.c.heads * a.q.group, rows * a.splits * a.waves / 4);
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
