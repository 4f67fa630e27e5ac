// What the block cache's attention kernels share (cache_attn.hip, 8 bits; cache4_attn.hip, 4 bits): which tokens a request's
// queries see, sums and maxima across lanes, the joining of a workgroup's waves.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "cache.h"
#include "cache_common.h"

namespace karpo {

constexpr int kAttendWaves = 4;
constexpr int kAttendThreads = 64 * kAttendWaves;

// Elements of the output that the waves join at once, and their sums' bytes (in the keys' array, when the groups are done).
constexpr int slab_of(int d, int nt) { return nt == 1 && d > 64 ? d / 2 : d / 4 > 32 ? d / 4 : 32; }
constexpr int sums_bytes(int d, int nt) { return kAttendWaves * 16 * nt * (slab_of(d, nt) + 4) * 4; }


struct Seen {
  int tokens, row, queries;  // cached tokens; first query row; query rows
  int first, groups;         // first group of 32 tokens that a query sees, and how many up to the last token
  int units;                 // groups, or 1 where there are queries and no tokens (their rows are zeros)
};

__device__ __forceinline__ Seen seen_of(const AttendParams& p, int i) {
  Seen s;
  s.tokens = min(max(p.r.lengths[i], 0), p.r.most);
  const int a = p.q_cu[i], b = p.q_cu[i + 1];
  s.row = a;
  s.queries = a >= 0 && b > a && b <= p.total_q ? b - a : 0;
  const int64_t before = (int64_t)s.tokens - s.queries - p.left;
  s.first = p.left >= 0 && before > 0 ? (int)(before < s.tokens ? before : s.tokens) / kCacheGroup : 0;
  s.groups = (s.tokens + kCacheGroup - 1) / kCacheGroup - s.first;
  s.units = s.queries > 0 ? max(s.groups, 1) : 0;
  return s;
}

// NaN into a request's rows past max_q, which nothing computes, of the key/value head's query heads (by the workgroups of its
// first vectors; here, at the attention kernel's end or in the join, it costs that kernel's loop no registers).
template <int D>
__device__ __forceinline__ void fill_past(const AttendParams& p, const Seen& s, int y, int first, int step) {
  if (s.queries > p.max_q && y < p.c.kv_heads)
    fill_rows<D>(kNanPair, p.o + (s.row + (int64_t)p.max_q) * p.so_t + (int64_t)y * p.group * p.so_h, p.so_t,
                 p.so_h, s.queries - p.max_q, p.group, first, step);
}

// A vector's position among its request's queries: vec / group, exactly (vec + 1/2 is no multiple of the group, and below
// 2^16 further from one than the product's rounding).
__device__ __forceinline__ int position_of(int vec, const AttendParams& p) { return (int)((vec + 0.5f) * p.per_group); }

// x's maximum / sum over the four lanes of a column (16 apart).
__device__ __forceinline__ float column_max(float x) {
  x = half_swap_max(x);
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __builtin_elementwise_maximum(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float column_sum(float x) {
  x = half_swap_sum(x);
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Two fp32 as packed bf16, in one instruction.
__device__ __forceinline__ unsigned pair_of(float a, float b) {
  return __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2{a, b}), bf16x2));
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}

// A barrier for what goes through LDS: copies and stores stay in flight.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

}  // namespace karpo
