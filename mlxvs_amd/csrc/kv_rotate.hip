// Queries and keys rotated by their tokens' positions, with or without a norm of
// each head in the same pass.
//
//   x' = x rsqrt(mean(x^2) + eps) w          (with a norm; over the whole head)
//   (a, b) -> magnitude (a cos t - b sin t, b cos t + a sin t),  t = position x frequency
//
// for the pairs (a, b) of the first `rotated` values: (x_2i, x_2i+1), or (x_i,
// x_i+rotated/2); the others pass.  An angle is a whole number: a frequency is kept
// as turns a position in 2^-64 of a turn, whose product with the position, modulo
// 2^64, is the exact fraction of a turn (the turns' own rounding makes 2^-33 of a turn
// at position 2^31, that of a frequency near 1 radian as a double 2^-25.6; in float32 an
// angle of 10^6 is off by 0.06).  The fraction is rounded to float32, by up to 2^-26 of
// a turn, for its sine and cosine.  All values are computed in float32 and rounded once.
//
// It moves bytes: every value is read once and written once, by loads that leave the
// caches alone (nontemporal: 43.6 -> 37.2 us with norms; stores like that are faster
// there, 35.7, but not without, 96 instead of 72).  Sines are made once for a (token,
// pair) and serve all heads.  Measured, 40 heads of 128 values: 16,001 tokens 72 us
// (4.5 TB/s both ways, a large copy 4.95), 8,192 with norms 37 us (4.5); 64 tokens
// 4.4 us of the GPU's time.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "kv_cache.h"
#include "kv_values.h"

namespace mlxvs::kern {
namespace {

// The cosine and sine of a position's angle, by magnitude.
__device__ __forceinline__ void turn(const KvRotateArgs& a, int64_t pos, int pair, float& c,
                                     float& s) {
  const uint64_t phase = (uint64_t)pos * a.turns[pair];
  // (the instructions take turns; a signed fraction keeps small angles' bits)
  const float x = (float)(int32_t)(phase >> 32) * 0x1p-32f;
#if defined(__HIP_DEVICE_COMPILE__)
  c = __builtin_amdgcn_cosf(x) * a.magnitude;
  s = __builtin_amdgcn_sinf(x) * a.magnitude;
#else
  c = s = x;
#endif
}

// A token's position in its text: what its request's cache lost counts too.
__device__ __forceinline__ int64_t text_position(const KvRotateArgs& a, int64_t t) {
  const int64_t pos = a.positions[t];
  if (pos < 0) return 0;  // (padding: turned by nothing)
  if (!a.evicted) return pos;
  const int r = a.token_request[t];
  return r >= 0 && r < a.requests ? pos + a.evicted[r] : pos;
}

template <bool BF16>
__device__ __forceinline__ uint16_t rounded(float x) {
  if constexpr (BF16) return __builtin_bit_cast(uint16_t, (__bf16)x);
  else return __builtin_bit_cast(uint16_t, (_Float16)x);
}

__device__ __forceinline__ float weight_at(const KvRows& r, bool bf16, int e) {
  if (r.norm_f32) return ((const float*)r.norm)[e];
  const uint16_t x = ((const uint16_t*)r.norm)[e];
  return bf16 ? value<true>(x) : value<false>(x);
}

// A lane's 16 weights of a norm.
template <bool BF16>
__device__ __forceinline__ void weights(const KvRows& r, int e0, int e1, bool on0, bool on1,
                                        float (&w)[16]) {
  typedef float floatx4 __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int e = half ? e1 : e0;
    const bool on = r.norm && (half ? on1 : on0);
    if (r.norm_f32) {
      floatx4 x[2] = {};
      if (on) {
        x[0] = *(const floatx4*)((const float*)r.norm + e);
        x[1] = *(const floatx4*)((const float*)r.norm + e + 4);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) w[8 * half + i] = x[i / 4][i % 4];
    } else {
      uintx4 x = {};
      if (on) x = *(const uintx4*)((const uint16_t*)r.norm + e);
#pragma unroll
      for (int i = 0; i < 8; ++i) w[8 * half + i] = value<BF16>(x, i);
    }
  }
}

// Any `rotated`: a wavefront a (token, head), a value a lane.  Loads of two bytes, twice
// for each value, and sines anew for each head: 8,192 tokens of 40 heads of 80 values, 40
// of them turned, 101 us (31 with 48 by the kernel below), with norms 143 (33).
template <bool BF16>
__global__ __launch_bounds__(256) void kv_rotate_any_kernel(KvRotateArgs a) {
  constexpr int kPer = kKvMaxDim / 64;
  const int lane = threadIdx.x & 63, heads = a.q.heads + a.k.heads;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t t = unit / heads;
  if (t >= a.tokens) return;
  const int i = (int)(unit % heads);
  const KvRows& r = i < a.q.heads ? a.q : a.k;
  const int h = i < a.q.heads ? i : i - a.q.heads;
  const uint16_t* x = (const uint16_t*)r.x + t * r.token + h * r.head;
  uint16_t* out = (uint16_t*)r.out + t * r.out_token + h * r.out_head;
  const int half = a.rotated / 2;
  float own[kPer], other[kPer], sum = 0.0f;
  int mate[kPer];
#pragma unroll
  for (int p = 0; p < kPer; ++p) {
    const int e = lane + 64 * p;
    mate[p] = a.pairs ? e ^ 1 : (e < half ? e + half : e - half);
    own[p] = e < a.dim ? value<BF16>(x[e]) : 0.0f;
    other[p] = e < a.rotated ? value<BF16>(x[mate[p]]) : 0.0f;
    sum += own[p] * own[p];
  }
  if (r.norm) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) sum += __shfl_xor(sum, m);
    const float inv = rsqrtf(sum / (float)a.dim + a.eps);
#pragma unroll
    for (int p = 0; p < kPer; ++p) {
      const int e = lane + 64 * p;
      if (e < a.dim) own[p] *= inv * weight_at(r, BF16, e);
      if (e < a.rotated) other[p] *= inv * weight_at(r, BF16, mate[p]);
    }
  }
  const int64_t pos = text_position(a, t);
  // (`out` may be `x`: all lanes' values are there before the first is written)
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int p = 0; p < kPer; ++p) {
    const int e = lane + 64 * p;
    if (e >= a.dim) continue;
    float y = own[p];
    if (e < a.rotated) {
      float c, s;
      turn(a, pos, a.pairs ? e / 2 : min(e, mate[p]), c, s);
      y = e < mate[p] ? y * c - other[p] * s : y * c + other[p] * s;
    }
    out[e] = rounded<BF16>(y);
  }
}

// `rotated` a multiple of 16 (a value a lane is 300 instead of 72 us, above): a lane has
// 16 values of a head, two pieces of 16 bytes that are turned with one another (halves)
// or within themselves (pairs), or that pass.  LANES lanes have a head, a wavefront
// 64 / LANES heads of one token at a time, with the same angles for all of them.
template <bool BF16, bool PAIRS, bool NORM, int LANES>
__global__ __launch_bounds__(256) void kv_rotate_kernel(KvRotateArgs a, int parts) {
  constexpr int kHeads = 64 / LANES, kAhead = 4;
  const int lane = threadIdx.x & 63, sub = lane % LANES, row = lane / LANES;
  const int64_t unit = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t t = unit / parts;
  if (t >= a.tokens) return;
  const int turned = a.rotated / 16;
  const bool turns = sub < turned;
  const int e0 = turns ? (PAIRS ? 16 : 8) * sub : 16 * sub;
  const int e1 = turns && !PAIRS ? e0 + a.rotated / 2 : e0 + 8;
  const bool on0 = e0 < a.dim, on1 = e1 < a.dim;
  // sets of heads, q's and then k's: kAhead of them are on their way at a time
  const int part = (int)(unit % parts), q_sets = (a.q.heads + kHeads - 1) / kHeads;
  const int sets = q_sets + (a.k.heads + kHeads - 1) / kHeads;
  uintx4 v[kAhead][2];
  const auto rows = [&](int set) -> const KvRows& { return set < q_sets ? a.q : a.k; };
  const auto head = [&](int set) { return (set < q_sets ? set : set - q_sets) * kHeads + row; };
  const auto load = [&](int first) {
#pragma unroll
    for (int n = 0; n < kAhead; ++n) {
      const int set = first + n * parts;
      v[n][0] = v[n][1] = uintx4{};
      if (set >= sets) continue;
      const KvRows& r = rows(set);
      const uint16_t* x = (const uint16_t*)r.x + t * r.token + head(set) * r.head;
      const bool there = head(set) < r.heads;
      if (there && on0) v[n][0] = __builtin_nontemporal_load((const uintx4*)(x + e0));
      if (there && on1) v[n][1] = __builtin_nontemporal_load((const uintx4*)(x + e1));
    }
  };
  float wq[16], wk[16];
  if constexpr (NORM) {
    weights<BF16>(a.q, e0, e1, on0, on1, wq);
    weights<BF16>(a.k, e0, e1, on0, on1, wk);
  }
  float c[8], s[8];
  const int64_t pos = text_position(a, t);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    c[i] = 1.0f;
    s[i] = 0.0f;
    if (turns) turn(a, pos, 8 * sub + i, c[i], s[i]);
  }
  for (int first = part; first < sets; first += kAhead * parts) {
    load(first);
#pragma unroll
    for (int n = 0; n < kAhead; ++n) {
      const int set = first + n * parts;
      if (set >= sets) continue;
      const KvRows& r = rows(set);
      float y[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) y[i] = value<BF16>(v[n][i / 8], i % 8);
      if constexpr (NORM) {
        if (r.norm) {
          float sum = 0.0f;
#pragma unroll
          for (int i = 0; i < 16; ++i) sum = fmaf(y[i], y[i], sum);
#pragma unroll
          for (int m = LANES / 2; m >= 1; m >>= 1) sum += __shfl_xor(sum, m);
          const float inv = rsqrtf(sum / (float)a.dim + a.eps);
#pragma unroll
          for (int i = 0; i < 16; ++i) y[i] *= inv * (set < q_sets ? wq[i] : wk[i]);
        }
      }
      if (turns) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int at = PAIRS ? 2 * i : i, with = PAIRS ? 2 * i + 1 : i + 8;
          const float u = y[at], z = y[with];
          y[at] = fmaf(u, c[i], -(z * s[i]));
          y[with] = fmaf(z, c[i], u * s[i]);
        }
      }
      uintx4 to[2];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        to[i / 4][i % 4] = rounded<BF16>(y[2 * i]) | (uint32_t)rounded<BF16>(y[2 * i + 1]) << 16;
      uint16_t* out = (uint16_t*)r.out + t * r.out_token + head(set) * r.out_head;
      const bool there = head(set) < r.heads;
      if (there && on0) *(uintx4*)(out + e0) = to[0];
      if (there && on1) *(uintx4*)(out + e1) = to[1];
    }
  }
}

int lanes_of(const KvRotateArgs& a) { return a.dim <= 64 ? 4 : a.dim <= 128 ? 8 : 16; }

// Wavefronts that share a token's heads: one where there are tokens enough (16,001
// and 8,192 tokens by one and four: 72 and 97 us, 37 and 62), as many as there are
// sets of heads where there are few.
int parts_of(const KvRotateArgs& a) {
  const int heads = 64 / lanes_of(a);
  const int64_t sets = (a.q.heads + heads - 1) / heads + (a.k.heads + heads - 1) / heads;
  return (int)std::max<int64_t>(1, std::min<int64_t>(sets, 4096 / a.tokens));
}

template <bool BF16, bool PAIRS, bool NORM>
void launch_lanes(const KvRotateArgs& a, dim3 grid, int parts, hipStream_t s) {
  switch (lanes_of(a)) {
    case 4: kv_rotate_kernel<BF16, PAIRS, NORM, 4><<<grid, 256, 0, s>>>(a, parts); break;
    case 8: kv_rotate_kernel<BF16, PAIRS, NORM, 8><<<grid, 256, 0, s>>>(a, parts); break;
    default: kv_rotate_kernel<BF16, PAIRS, NORM, 16><<<grid, 256, 0, s>>>(a, parts);
  }
}

template <bool BF16>
void launch_type(const KvRotateArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)kv_rotate_grid(a));
  if (a.rotated % 16) {
    kv_rotate_any_kernel<BF16><<<grid, 256, 0, s>>>(a);
    return;
  }
  const int parts = parts_of(a);
  const bool norm = a.q.norm || a.k.norm;
  if (a.pairs) norm ? launch_lanes<BF16, true, true>(a, grid, parts, s) : launch_lanes<BF16, true, false>(a, grid, parts, s);
  else norm ? launch_lanes<BF16, false, true>(a, grid, parts, s) : launch_lanes<BF16, false, false>(a, grid, parts, s);
}

}  // namespace

int64_t kv_rotate_grid(const KvRotateArgs& a) {
  if (a.tokens == 0) return 0;
  if (a.rotated % 16) return (a.tokens * (a.q.heads + a.k.heads) + 3) / 4;
  return (a.tokens * parts_of(a) + 3) / 4;
}

hipError_t launch_kv_rotate(const KvRotateArgs& a, hipStream_t s) {
  a.bf16 ? launch_type<true>(a, s) : launch_type<false>(a, s);
  return hipGetLastError();
}

}  // namespace mlxvs::kern
