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

// The maximum over the lanes of one column (l, l ^ 16, l ^ 32, l ^ 48).
__device__ __forceinline__ float column_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float column_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
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

// DP: head size rounded up to a multiple of 32.  LIST: over listed blocks.  P16:
// pages of 16 keys, two to a 32-key pair.
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
    const int ps = a.c.page, lps = a.c.lps;
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
          if (32 * i + 8 * grp < d) kf[2 * p + u][i] = *(const uintx4*)(kp[p] + 4 * u * d + 32 * i);
        }
#pragma unroll
    for (int p = 0; p < kPairs; ++p)
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        vf[p][i] = uintx4{};
        if (16 * i + col < d) vf[p][i] = *(const uintx4*)(vp[p] + 16 * i * ps);
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

// Many rows: a wavefront each, no parts.
constexpr int64_t kManyRows = 4096;

template <int DP, bool BF16, bool LIST, bool P16>
__global__ __launch_bounds__(256, 2) void kv_attend_rows_kernel(KvAttendArgs a) {
  using A = Attend<DP, BF16, LIST, P16>;
  const int tiles = (a.q.group + kColumns - 1) / kColumns;
  const int64_t row = blockIdx.x;
  const int mt = (int)(row % tiles);
  const int h = (int)(row / tiles % a.c.heads);
  const int64_t t = row / tiles / a.c.heads * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (t >= a.q.tokens) return;
  A w(a, threadIdx.x & 63);
  w.start(t, h, mt);
  const int r = a.q.token_request[t], pos = a.q.positions[t];
  if (r >= 0 && r < a.q.requests && pos >= 0) {
    const int end = LIST ? a.n : min(pos >> a.c.lps, a.q.cols - 1) + 1;
    for (int e = 0; e < end; e += 64) {
      w.entries(t, h, r, pos, e, end);
      const int64_t k1 = (int64_t)min(end, e + 64) << a.c.lps;
      for (int64_t k = (int64_t)e << a.c.lps; k < k1; k += A::kKeys) w.step(h, (int)k);
    }
  }
  const float l = column_sum(w.l);
  const int g = mt * kColumns + w.col;
  if (g >= a.q.group) return;
  const float inv = 1.0f / l;
  const int64_t at = t * a.c.heads * a.q.group + h * a.q.group + g;
#pragma unroll
  for (int i = 0; i < A::kTiles; ++i) {
    const int d = 16 * i + 4 * w.grp;
    if (d < a.c.dim) {
      typename A::Tx4 x;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = (typename A::T)(l == 0.0f ? 0.0f : w.o[i][j] * inv);
      *(typename A::Tx4*)((typename A::T*)a.out + at * a.c.dim + d) = x;
    }
  }
  if (a.lse && w.grp == 0) a.lse[at] = lse_of(w.m, l, a.scale, A::kBias);
}

// Few rows: a part of a row's keys for each workgroup, its steps dealt to the
// W wavefronts in turn.
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

template <int DP, bool BF16, bool LIST, bool P16>
void launch_one(const KvAttendArgs& a, hipStream_t s) {
  const int tiles = (a.q.group + kColumns - 1) / kColumns;
  if (a.waves == 1) {
    const int64_t grid = (a.q.tokens + 3) / 4 * a.c.heads * tiles;
    kv_attend_rows_kernel<DP, BF16, LIST, P16><<<dim3((unsigned)grid), 256, 0, s>>>(a);
  } else {
    const dim3 grid((unsigned)(a.q.tokens * a.c.heads * tiles * a.splits));
    if (a.waves == 8) kv_attend_parts_kernel<DP, BF16, LIST, P16, 8><<<grid, 512, 0, s>>>(a);
    else kv_attend_parts_kernel<DP, BF16, LIST, P16, 4><<<grid, 256, 0, s>>>(a);
  }
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
  if (rows >= kManyRows) {
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
  return std::max(a.q.tokens * a.c.heads * a.q.group,
                  (a.q.tokens + 3) * a.c.heads * ((a.q.group + kColumns - 1) / kColumns) * a.splits);
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
