// Queries and keys rotated by their tokens' positions, with or without a norm of
// each head in the same pass.
//
//   x' = x rsqrt(mean(x^2) + eps) w          (with a norm; over the whole head)
//   (a, b) -> magnitude (a cos t - b sin t, b cos t + a sin t),  t = position x frequency
//
// for the pairs (a, b) of the first `rotated` values: (x_2i, x_2i+1), or (x_i,
// x_i+rotated/2); the others pass.  An angle is a whole number: a frequency is kept
// as turns a position in 2^-64 of a turn, whose product with the position, modulo
// 2^64, is the exact fraction of a turn (a frequency's rounding makes 2^-33 of a
// turn at position 2^31; in float32 an angle of 10^6 is off by 0.06).  All
// values are computed in float32 and rounded once.
//
// It moves bytes: every value is read once and written once.  Sines are made once
// for a (token, pair) and serve all heads.
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
  if (pos < 0) return 0;  // (padding: not rotated)
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

// Any `rotated`: a wavefront a (token, head), a value a lane.
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

}  // namespace

int64_t kv_rotate_grid(const KvRotateArgs& a) {
  return (a.tokens * (a.q.heads + a.k.heads) + 3) / 4;
}

hipError_t launch_kv_rotate(const KvRotateArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)kv_rotate_grid(a));
  if (a.bf16) kv_rotate_any_kernel<true><<<grid, 256, 0, s>>>(a);
  else kv_rotate_any_kernel<false><<<grid, 256, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace mlxvs::kern
