// Device helpers of the block cache's kernels.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mfma_common.h"

namespace karpo {

typedef float f32x2 __attribute__((ext_vector_type(2)));

__host__ __device__ __forceinline__ int64_t ka_min64(int64_t a, int64_t b) { return a < b ? a : b; }

// 2^e, -126 <= e <= 127.
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }

// Two e4m3 codes of `w` (its upper two with `up`) times `scale` (a power of two: exact) as packed bf16.
__device__ __forceinline__ unsigned bf16_pair(unsigned w, float scale, bool up) {
  return up ? __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true))
            : __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false));
}
__device__ __forceinline__ u32x4 bf16_of_8(unsigned a, unsigned b, float scale) {
  return u32x4{bf16_pair(a, scale, false), bf16_pair(a, scale, true), bf16_pair(b, scale, false),
               bf16_pair(b, scale, true)};
}

constexpr unsigned kNanPair = 0x7fc07fc0u;  // two bf16

// Pairs `x` into `count` rows of `heads` heads from o on, by threads `first`, `first` + `step`, ...
template <int D>
__device__ __forceinline__ void fill_rows(unsigned x, uint16_t* o, int64_t s_row, int64_t s_head, int64_t count, int heads,
                                          int64_t first, int64_t step) {
  for (int64_t e = first; e < count * heads * (D / 8); e += step) {
    const int64_t vec = e / (D / 8), row = vec / heads;
    *reinterpret_cast<u32x4*>(o + row * s_row + (vec - row * heads) * s_head + e % (D / 8) * 8) =
        u32x4{x, x, x, x};
  }
}

// The sum over the wave's lanes up to this one, in registers (six additions across lanes, no LDS).
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // from the lane 1, 2, 4, 8 before, within 16
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // lane 15 of the row of 16 before, into rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // lane 31, into rows 2 and 3
  return x;
}

// v: the sum over the workgroup's threads before this one, of N values; all: over all of them. `part` is free again after
// the caller's next barrier.
template <int THREADS, int N>
__device__ __forceinline__ void block_scan(int (&v)[N], int (&all)[N], int (*part)[N]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int own[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    own[k] = v[k];
    v[k] = wave_scan(v[k]);
    if (lane == 63) part[wave][k] = v[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) {
    int before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
      const int t = part[w][k];
      if (w < wave) before += t;
      sum += t;
    }
    v[k] += before - own[k];
    all[k] = sum;
  }
}

// The last j < n with first[j] <= x (first[0] <= x, non-decreasing).
__device__ __forceinline__ int last_at_most(const int* first, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

}  // namespace karpo
