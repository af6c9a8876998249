// The n tokens of each request and kv head that a budget leaves: the first and
// the recent ones, and of the others those of the largest mass, the lowest among
// equal ones, in their order.  A request of at most `above` tokens keeps all: its
// list is empty.
//
// Masses are compared as 32-bit ranks in their order (NaN last), so the list is a
// matter of definition.  The n-th largest rank is found by 11, 11 and 10 of its
// bits, a histogram of 2,048 bins in LDS each; then the tokens above it are taken,
// and the first of those that equal it.
//
// A row of up to 32,768 slots is a workgroup's and read once: its ranks stay in
// registers; so is one of up to 65,536 where there are more than 64 rows.  Others are
// split into parts of 8,192 or more, a workgroup each, with a launch for every histogram
// and one for the list: the parts' histograms are summed by whoever needs them, so that
// nothing is counted by atomics in memory.  (With 64 ranks a lane, rows of more than
// 32,768 slots and parts of rows of more than 1,048,576, not all stay in registers: 33 to
// 76 of 128 are spilled.)
//
// Chains of small steps, far from the bytes' 2 us: 256 rows of 16,384 slots 15 us (53
// if all masses are equal, whose counts meet in one place; 20 if half of them are), 8
// rows of 262,144 33 us (53) in four launches of 5, 11, 10 and 10: each workgroup of the
// later ones sums all parts' histograms.
#include <hip/hip_runtime.h>

#include "kv_cache.h"

namespace mlxvs::kern {
namespace {

constexpr uint32_t kAlways = 0xFFFFFFFFu;
constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBins = 2048, kDigits = 3;

__device__ __forceinline__ int shift_of(int digit) { return digit == 0 ? 21 : digit == 1 ? 10 : 0; }
__device__ __forceinline__ int bins_of(int digit) { return digit == 2 ? 1024 : kBins; }
__device__ __forceinline__ uint32_t digit_of(uint32_t rank, int digit) {
  return digit == 2 ? rank & 1023 : rank >> shift_of(digit) & 2047;
}

__device__ __forceinline__ int bits(uint64_t x) { return (int)__popcll(x); }

// A mass as a rank: greater masses, greater ranks; -0 and 0 are equal, NaN is 1
// (below minus infinity), 0 stands for no token.
__device__ __forceinline__ uint32_t rank_of(float x) {
  if (x != x) return 1;
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);
  return u >> 31 ? ~u : u | 0x80000000u;
}

// Ranks of 64 R tokens from `from` on for each wavefront, 64 neighbours at a time.
template <int R>
struct Ranks {
  uint32_t k[R];
  int from;  // this lane's first token

  // (read first, ranked once something else has been read, too)
  __device__ __forceinline__ Ranks(const float* mass, int start, int length) {
    from = start + (threadIdx.x >> 6) * 64 * R + (threadIdx.x & 63);
#pragma unroll
    for (int i = 0; i < R; ++i)
      k[i] = __builtin_bit_cast(uint32_t, from + 64 * i < length ? mass[from + 64 * i] : 0.0f);
  }
  __device__ __forceinline__ void rank(const KvKeepArgs& a, int length) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int t = from + 64 * i;
      k[i] = t >= length                             ? 0
             : t < a.first || t >= length - a.recent ? kAlways
                                                     : rank_of(__builtin_bit_cast(float, k[i]));
    }
  }

  // Counts those whose higher digits are prefix's in hist.
  __device__ __forceinline__ void count(uint32_t* hist, int digit, uint32_t prefix) const {
    const uint32_t known = digit == 0 ? 0 : ~0u << shift_of(digit - 1);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (k[i] != 0 && (k[i] & known) == prefix) atomicAdd(&hist[digit_of(k[i], digit)], 1u);
    }
  }

  // The tokens above `cut`, and of those that equal it the first `ties` of the
  // workgroup, into out in their order.
  __device__ __forceinline__ void take(uint32_t cut, int ties, int32_t* out, int (*waves)[2]) const {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int gt = 0, eq = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      gt += bits(__ballot(k[i] > cut));
      eq += bits(__ballot(k[i] == cut));
    }
    if (lane == 0) {
      waves[wave][0] = gt;
      waves[wave][1] = eq;
    }
    __syncthreads();
    int at = 0, before = 0;
    for (int w = 0; w < wave; ++w) {
      at += waves[w][0] + min(waves[w][1], max(0, ties - before));
      before += waves[w][1];
    }
    const uint64_t below = (uint64_t(1) << lane) - 1;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const uint64_t tied = __ballot(k[i] == cut);
      const bool taken = k[i] > cut || (k[i] == cut && before + bits(tied & below) < ties);
      const uint64_t all = __ballot(taken);
      if (taken) out[at + bits(all & below)] = from + 64 * i;
      at += bits(all);
      before += bits(tied);
    }
  }
};

struct Pick {
  int waves[kWaves];
  uint32_t bin;
  int left;
};

// The bin in which the left-th largest lies, and the how manieth it is there, from
// this thread's two bins (counted from the largest: thread i has 2047 - 2 i and the
// one below).
__device__ __forceinline__ void pick(int hi, int lo, int left, Pick& s) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int upto = hi + lo;
#pragma unroll
  for (int by = 1; by < 64; by <<= 1) {
    const int y = __shfl_up(upto, by);
    if (lane >= by) upto += y;
  }
  if (lane == 63) s.waves[wave] = upto;
  __syncthreads();
  for (int w = 0; w < wave; ++w) upto += s.waves[w];
  const int before = upto - hi - lo;
  if (before < left && left <= upto) {
    const bool upper = left <= before + hi;
    s.bin = kBins - 1 - 2 * threadIdx.x - (upper ? 0 : 1);
    s.left = left - before - (upper ? 0 : hi);
  }
  __syncthreads();
}

__device__ __forceinline__ int length_of(const KvKeepArgs& a, int64_t row) {
  return (int)min<int64_t>(a.lengths[row / a.heads], a.slots);
}

__device__ __forceinline__ void none(const KvKeepArgs& a, int32_t* out) {
  for (int i = threadIdx.x; i < a.n; i += kThreads) out[i] = -1;
}

// A row a workgroup, of up to 1,024 R slots.
template <int R>
__global__ __launch_bounds__(kThreads) void kv_keep_kernel(KvKeepArgs a) {
  __shared__ uint32_t hist[kBins];
  __shared__ Pick s;
  __shared__ int waves[kWaves][2];
  const int64_t row = blockIdx.x;
  const int length = length_of(a, row), tid = threadIdx.x;
  int32_t* out = a.kept + row * a.n;
  if (length <= a.above) return none(a, out);
  Ranks<R> ranks(a.mass + row * a.slots, 0, length);
  ranks.rank(a, length);
  uint32_t cut = 0;
  int left = a.n;
#pragma unroll 1
  for (int digit = 0; digit < kDigits; ++digit) {
    hist[tid] = hist[tid + kThreads] = 0;
    __syncthreads();
    ranks.count(hist, digit, cut);
    __syncthreads();
    pick((int)hist[kBins - 1 - 2 * tid], (int)hist[kBins - 2 - 2 * tid], left, s);
    cut |= s.bin << shift_of(digit);
    left = s.left;
    if (left == (int)hist[s.bin] && cut != 0 && digit + 1 < kDigits) {
      // all of the bin are taken: those above the rank below it
      cut -= 1;
      left = 0;
      break;
    }
    __syncthreads();
  }
  ranks.take(cut, left, out, waves);
}

// ---- rows in parts ----------------------------------------------------------------

// The workspace, for each row and part: a histogram for each digit, how many of it
// are above the digits known; for each row: those digits and how many are left.
struct Work {
  uint32_t* hist;  // [rows][parts][3][2048]
  int* above;      // [rows][parts][2]: by the first digit, by the second
  uint32_t* known; // [rows][2][2]: after the first and second digit: prefix, left
};
// Slots of a part for each of its threads: few, but no more than 32 parts if that can
// be, since each reads the histograms of all.  8 rows of 262,144 slots with 4, 8, 16, 32:
// 59, 34, 37, 51 us; of 1,048,576 with 16, 32, 64: 97, 78, 139.
__host__ __device__ __forceinline__ int each_of(const KvKeepArgs& a) {
  int each = 8;
  while (each < 64 && a.slots > (int64_t)32 * kThreads * each) each *= 2;
  return each;
}
__host__ __device__ __forceinline__ int64_t parts_of(const KvKeepArgs& a) {
  const int part = kThreads * each_of(a);
  return (a.slots + part - 1) / part;
}
__device__ __forceinline__ Work work_of(const KvKeepArgs& a) {
  const int64_t rows = a.requests * a.heads, units = rows * parts_of(a);
  uint32_t* w = (uint32_t*)a.work;
  return {w, (int*)(w + units * kDigits * kBins), w + units * (kDigits * kBins + 2)};
}

// STEP 0, 1, 2: the part's histogram of that digit, the one before it being found
// first.  STEP 3: the list.
template <int STEP, int R>
__global__ __launch_bounds__(kThreads) void kv_keep_part_kernel(KvKeepArgs a) {
  constexpr int kPart = kThreads * R;
  __shared__ uint32_t hist[kBins];
  __shared__ Pick s;
  __shared__ int waves[kWaves][2];
  __shared__ int sums[kWaves], same;
  const int parts = (int)parts_of(a), tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x / parts;
  const int part = (int)(blockIdx.x % parts), length = length_of(a, row);
  int32_t* out = a.kept + row * a.n;
  if (length <= a.above) {
    if (STEP == 3 && part == 0) none(a, out);
    return;
  }
  const int some = (length - 1) / kPart + 1;  // parts that hold tokens
  if (part >= some) return;
  const Work work = work_of(a);
  Ranks<R> ranks(a.mass + row * a.slots, part * kPart, length);
  if (STEP == 0) ranks.rank(a, length);
  const auto hist_of = [&](int p, int digit) {
    return work.hist + ((row * parts + p) * kDigits + digit) * kBins;
  };
  uint32_t prefix = 0;
  int left = a.n;
  const int b0 = kBins - 2 - 2 * tid;  // this thread's bins: b0 + 1, b0
  if constexpr (STEP > 0) {
    constexpr int kDigit = STEP - 1;
    if constexpr (STEP > 1) {
      prefix = work.known[row * 4 + (STEP - 2) * 2];
      left = (int)work.known[row * 4 + (STEP - 2) * 2 + 1];
    }
    int hi = 0, lo = 0;  // over all parts; and of this one, or for the list of those before it
    int hi_here = 0, lo_here = 0;
    if (b0 < bins_of(kDigit)) {
#pragma unroll 16
      for (int p = 0; p < some; ++p) {
        const uint2 x = *(const uint2*)(hist_of(p, kDigit) + b0);
        lo += (int)x.x;
        hi += (int)x.y;
        if (STEP == 3 ? p < part : p == part) {
          lo_here += (int)x.x;
          hi_here += (int)x.y;
        }
      }
    }
    ranks.rank(a, length);
    pick(hi, lo, left, s);
    const uint32_t bin = s.bin;
    prefix |= bin << shift_of(kDigit);
    left = s.left;
    // how many of those are above the bin
    const int over = (b0 + 1 > (int)bin ? hi_here : 0) + (b0 > (int)bin ? lo_here : 0);
    const auto total = [&](int x) {
#pragma unroll
      for (int i = 32; i >= 1; i >>= 1) x += __shfl_xor(x, i);
      if (lane == 0) sums[wave] = x;
      __syncthreads();
      x = 0;
      for (int w = 0; w < kWaves; ++w) x += sums[w];
      return x;
    };
    if constexpr (STEP < 3) {
      const int mine = total(over);
      if (tid == 0) {
        work.above[(row * parts + part) * 2 + kDigit] = mine;
        if (part == 0) {
          work.known[row * 4 + kDigit * 2] = prefix;
          work.known[row * 4 + kDigit * 2 + 1] = (uint32_t)left;
        }
      }
    } else {
      // where this part's tokens go: after those of the parts before it
      int gt = over;
      for (int p = tid; p < part; p += kThreads)
        gt += work.above[(row * parts + p) * 2] + work.above[(row * parts + p) * 2 + 1];
      if (b0 == (int)bin || b0 + 1 == (int)bin) same = b0 == (int)bin ? lo_here : hi_here;
      gt = total(gt);
      const int eq = same;
      ranks.take(prefix, max(0, left - eq), out + gt + min(eq, left), waves);
      return;
    }
  }
  hist[tid] = hist[tid + kThreads] = 0;
  __syncthreads();
  ranks.count(hist, STEP, prefix);
  __syncthreads();
  uint2* to = (uint2*)hist_of(part, STEP);
  if (2 * tid < bins_of(STEP)) to[tid] = *(const uint2*)(hist + 2 * tid);
}

template <int STEP>
hipError_t launch_step(const KvKeepArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)kv_keep_grid(a));
  switch (each_of(a)) {
    case 8: kv_keep_part_kernel<STEP, 8><<<grid, kThreads, 0, s>>>(a); break;
    case 16: kv_keep_part_kernel<STEP, 16><<<grid, kThreads, 0, s>>>(a); break;
    case 32: kv_keep_part_kernel<STEP, 32><<<grid, kThreads, 0, s>>>(a); break;
    default: kv_keep_part_kernel<STEP, 64><<<grid, kThreads, 0, s>>>(a);
  }
  return hipGetLastError();
}

// Whether rows are split.  Whole / in parts: 8 rows of 32,768 slots 25 / 27 us, of
// 65,536 51 / 31; 64 rows of 65,536 53 / 45, 256 of them 68 / 150.
bool in_parts(const KvKeepArgs& a) {
  return a.slots > 65536 || (a.slots > 32768 && a.requests * a.heads <= 64);
}

}  // namespace

int64_t kv_keep_workspace(const KvKeepArgs& a) {
  if (!in_parts(a)) return 0;
  const int64_t rows = a.requests * a.heads;
  return 4 * (rows * parts_of(a) * (kDigits * kBins + 2) + 4 * rows);
}

int64_t kv_keep_grid(const KvKeepArgs& a) {
  return a.requests * a.heads * (in_parts(a) ? parts_of(a) : 1);
}

hipError_t launch_kv_keep(const KvKeepArgs& a, hipStream_t s) {
  if (!in_parts(a)) {
    const dim3 grid((unsigned)kv_keep_grid(a));
    if (a.slots <= 4096) kv_keep_kernel<4><<<grid, kThreads, 0, s>>>(a);
    else if (a.slots <= 16384) kv_keep_kernel<16><<<grid, kThreads, 0, s>>>(a);
    else if (a.slots <= 32768) kv_keep_kernel<32><<<grid, kThreads, 0, s>>>(a);
    else kv_keep_kernel<64><<<grid, kThreads, 0, s>>>(a);
    return hipGetLastError();
  }
  hipError_t e = launch_step<0>(a, s);
  if (e == hipSuccess) e = launch_step<1>(a, s);
  if (e == hipSuccess) e = launch_step<2>(a, s);
  if (e == hipSuccess) e = launch_step<3>(a, s);
  return e;
}

}  // namespace mlxvs::kern
