// The attention that each cached key gets: for every key p of a request and kv
// head, over the step's tokens t that see it and the head's query heads g,
//
//   mass_p = (p < first ? decay mass_p : 0) + sum_t sum_g exp(scale q_tg.k_p - lse_tg)
//
// with the logarithms of sums that attention over the same keys returned; first is
// the request's first new position, so that a key's mass starts with its own step.
// A key's sum has one owner and a fixed order: no atomics, the same bits every time.
//
// S = K Q^T on the matrix cores with the keys as rows: a wavefront keeps its keys'
// values in registers, the operand of every product, and goes through the tokens'
// query heads, 16 columns at a time.  A lane adds up its column's weights of each
// key over all of them, and the columns meet once at the end.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "kv_cache.h"
#include "kv_mfma.h"

namespace mlxvs::kern {
namespace {

constexpr int kTileKeys = 16, kTiles = 4;      // of a wavefront
constexpr int kWaveKeys = kTileKeys * kTiles;
constexpr int kChunk = 4 * kWaveKeys;          // keys of a workgroup

// A request's tokens of the step, and the keys that they see.
struct Span {
  int begin, tokens;
  int first, last;  // positions of the first and the last token
};

__device__ __forceinline__ Span span_of(const KvWeighArgs& a, int r) {
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

// The sum over the 16 lanes of a row.
__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
  for (int i = 8; i >= 1; i >>= 1) x += __shfl_xor(x, i);
  return x;
}

template <int DP, bool BF16>
__global__ __launch_bounds__(256, 2) void kv_weigh_kernel(KvWeighArgs a, int chunks) {
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
    const int k0 = (int)at + wave * kWaveKeys;
    if (k0 > sp.last) return;
    uintx4 kf[kTiles][kSteps];
    bool there[kTiles];
#pragma unroll
    for (int u = 0; u < kTiles; ++u) {
      const int k = k0 + kTileKeys * u;
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
    float sum[kTiles][4] = {};
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
      for (int u = 0; u < kTiles; ++u) {
        floatx4 s = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
          s = mfma(__builtin_bit_cast(Tx8, kf[u][i]), __builtin_bit_cast(Tx8, q[i]), s);
        const int seen = pos - (k0 + kTileKeys * u + 4 * grp);  // keys up to this one
#pragma unroll
        for (int i = 0; i < 4; ++i)
          sum[u][i] += i <= seen ? __builtin_amdgcn_exp2f(fmaf(s[i], a.scale, -lse) * kLog2e) : 0.0f;
      }
    }
#pragma unroll
    for (int u = 0; u < kTiles; ++u) {
      float mine = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float all = row_sum(sum[u][i]);
        if (col == i) mine = all;
      }
      const int p = k0 + kTileKeys * u + 4 * grp + col;
      if (col < 4 && p <= sp.last) {
        const float before = p < sp.first && a.decay != 0.0f ? a.decay * mass[p] : 0.0f;
        mass[p] = before + (there[u] ? mine : 0.0f);
      }
    }
  }
}

int64_t chunks_of(const KvWeighArgs& a) {
  const int64_t most = std::min<int64_t>(a.longest, (int64_t)a.q.cols << a.c.lps);
  return std::max<int64_t>(1, (most + kChunk - 1) / kChunk);
}

template <int DP, bool BF16>
void launch_dim(const KvWeighArgs& a, hipStream_t s) {
  kv_weigh_kernel<DP, BF16><<<dim3((unsigned)kv_weigh_grid(a)), 256, 0, s>>>(a, (int)chunks_of(a));
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

int64_t kv_weigh_grid(const KvWeighArgs& a) {
  return a.q.requests * a.c.heads * chunks_of(a);
}

hipError_t launch_kv_weigh(const KvWeighArgs& a, hipStream_t s) {
  a.c.bf16 ? launch_type<true>(a, s) : launch_type<false>(a, s);
  return hipGetLastError();
}

}  // namespace mlxvs::kern
