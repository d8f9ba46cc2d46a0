// Device helpers shared by the paged KV cache kernels (paged.cu, attention_paged.cu).
#pragma once

#include "common.cuh"
#include "paged_args.h"

namespace pai {
namespace paged {

// An integral F32 value in [lo, hi] (hi <= 2^24, which F32 holds exactly).
__device__ __forceinline__ bool integral(float f, int lo, int hi, int& out) {
  if (!(f >= (float)lo && f <= (float)hi) || f != floorf(f)) return false;
  out = (int)f;
  return true;
}

// Exact division of 0 <= x < 2^31 by d (a page size, the heads of a group): with 2^(l-1) < d <= 2^l and m = ceil(2^(31+l) / d) <= 2^32 - 1,
// x m / 2^(31+l) exceeds x / d by less than x 2^l / (d 2^(31+l)) < 1 / d, which reaches no further integer.
struct PageDiv {
  int size;
  unsigned mul;
  int shift;
  __device__ __forceinline__ int div(int x) const { return (int)(((uint64_t)(unsigned)x * mul) >> shift); }
};
inline PageDiv page_div(int size) {
  const uint64_t d = size > 0 ? size : 1;
  int l = 0;
  while (1ull << l < d) l++;
  return PageDiv{size, (unsigned)(((1ull << (31 + l)) + d - 1) / d), 31 + l};
}

inline bool aligned(const pai_tensor& t) {  // 16-byte rows: every index but the last moves by whole float4
  if (reinterpret_cast<uintptr_t>(fptr(t)) % 16) return false;
  for (int i = 0; i + 1 < t.rank; i++)
    if (t.dims[i] > 1 && t.strides[i] % 4) return false;
  return true;
}

// Exclusive prefix sums of N values per thread over the block, in thread order; totals in every thread. `tmp` holds N values
// per warp.
template <int THREADS, int N>
__device__ __forceinline__ void block_prefix(const int64_t (&v)[N], int64_t* tmp, int64_t (&before)[N], int64_t (&total)[N]) {
  static_assert(THREADS % 32 == 0 && THREADS <= 1024, "one value per lane for the warps' sums");
  constexpr int kWarps = THREADS / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t x[N];
#pragma unroll
  for (int k = 0; k < N; k++) x[k] = v[k];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
#pragma unroll
    for (int k = 0; k < N; k++) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x[k], o);
      if (lane >= o) x[k] += y;
    }
  }
  __syncthreads();  // tmp may still be read from an earlier call
#pragma unroll
  for (int k = 0; k < N; k++)
    if (lane == 31) tmp[k * kWarps + warp] = x[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; k++) {
    int64_t w = lane < kWarps ? tmp[k * kWarps + lane] : 0;  // every warp sums the warps' sums
#pragma unroll
    for (int o = 1; o < kWarps; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    total[k] = __shfl_sync(0xffffffffu, w, kWarps - 1);
    const int64_t warps = __shfl_sync(0xffffffffu, w, warp > 0 ? warp - 1 : 0);
    before[k] = (warp > 0 ? warps : 0) + x[k] - v[k];
  }
}

// a / b of numbers that are not negative; most fit 32 bits, whose division is several times shorter.
__device__ __forceinline__ int64_t div_pos(int64_t a, int64_t b) {
  if (((a | b) >> 32) == 0) return (uint32_t)a / (uint32_t)b;
  return a / b;
}

}  // namespace paged
}  // namespace pai
