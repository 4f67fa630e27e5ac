// Attention over the block cache for few queries per request (karpo_cache_attend): the keys of all requests are split evenly
// over the GPU, 32 tokens at a time, and the shares of a request joined by a second launch.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "cache.h"
#include "cache_common.h"

namespace karpo {

namespace {

constexpr int kAttendWaves = 4;
constexpr int kAttendThreads = 64 * kAttendWaves;
// Waves per SIMD (and workgroups per CU).
__host__ __device__ constexpr int attend_waves(int d, int nt) {
  return nt == 1 && d <= 128 ? 4 : d == 64 && nt == 2 ? 3 : d <= 128 || (d == 256 && nt == 1) ? 2 : 1;
}
// Bytes of LDS for the waves' copies of a group's keys (as many for the values).
constexpr int ring_bytes(int d) { return kAttendWaves * kCacheGroup * d; }
// Elements of the output that the waves join at once, and their sums' bytes (in the keys' array, when the groups are done).
constexpr int slab_of(int d, int nt) { return nt == 1 && d > 64 ? d / 2 : d / 4 > 32 ? d / 4 : 32; }
constexpr int sums_bytes(int d, int nt) { return kAttendWaves * 16 * nt * (slab_of(d, nt) + 4) * 4; }

// Requests of which at most this many tokens are seen are not split (a quarter of it at head size 512): one workgroup walks
// their groups, five a wave, and there is nothing to join. Split against whole, 8 requests: head size 64, 512 tokens 16.9,
// 12.8 us, 2,048 tokens 16.7, 21.6; 128, 768 tokens 16.7, 13.9, 1,024 tokens 16.6, 16.7; 256, 512 tokens 16.7, 14.5, 768
// tokens 16.6, 18.3; 512, 128 tokens 17.0, 13.3, 256 tokens 16.8, 18.0. 128 requests of 512 tokens at head size 128 49.6,
// 44.0; at 512 61.4, 60.7.
constexpr int64_t kWholeTokens = 640;
constexpr int kLeastUnits = kAttendWaves;  // groups of 32 tokens that a workgroup takes at least

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

// What a request takes of the sums: a workgroup that goes on to a next request spends about as long on the change (joining its
// waves, the new queries and tables, the first copies) as on kStart groups. Shares by groups alone left the last workgroups of
// 48 ragged requests 15 us behind the middle one.
constexpr int kStart = 4;
__device__ __forceinline__ int weight_of(int units) { return units > 0 ? units + kStart : 0; }

// The workgroups' shares of `total` units: of `parts` workgroups (fewer where each would get less than kLeastUnits) the first
// `more` take `each` + 1, the others `each`.
struct Shares {
  int each, more;
  __device__ __forceinline__ Shares(int total, int parts) {
    const unsigned n = max(min(parts, total / kLeastUnits), 1);
    each = (int)((unsigned)total / n);
    more = total - each * (int)n;
  }
  __device__ __forceinline__ int begin(int part) const { return part * each + min(part, more); }
  __device__ __forceinline__ int part_of(int unit) const {
    const int longer = more * (each + 1);
    return unit < longer ? (int)((unsigned)unit / (unsigned)(each + 1)) : more + (int)((unsigned)(unit - longer) / (unsigned)each);
  }
};

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

__device__ __forceinline__ bf16x8 operand(unsigned a, unsigned b, float scale) {
  return __builtin_bit_cast(bf16x8, bf16_of_8(a, b, scale));
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

// Which of a word's four codes are NaN, as 0x80 in their bytes.
__device__ __forceinline__ unsigned nan_codes(unsigned w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// One lane's view of a group of 32 tokens with 16x16x32 matrix instructions: S^T = K Q^T has the keys as rows (two tiles),
// the query vectors as columns: column lane % 16, keys 16 t + 4 (lane / 16) + i. Those are this lane's eight weights, and as
// they stand the second operand of O^T = V^T P^T, whose first operand, 8 of these keys of one element, is 8 bytes of the cache.
// The products are of bf16 operands (a cached element is one exactly); the weights enter as two bf16 terms, 2^-17 off, which
// costs matrix work that this kernel, bound by the codes' way from HBM, has to spare (2-norm error against 64 bits with
// one term and with two, the latter the output's own rounding: 2.31e-3, 1.67e-3 for one query over 131,073 tokens at head size
// 512; 1.04e-3, 0.81e-3 for 48 requests at 128; in time 91.2, 91.3 us and 48.8, 50.8 us).
//
// A wave takes every fourth group of its workgroup's share by itself, its running maximum and sums in registers, the next
// group's keys on their way to LDS while this one's weights are made, the next values while the next keys are read: a group in
// flight a wave (8 KiB at head size 128, four waves a SIMD; 32 KiB at 512, one). Registers for them instead of LDS spilled at
// head size 512: 240 us for one token over 131,072, 119 with LDS. Nothing but a request's end joins the waves.
//
// Measured (codes read / time of this kernel): 48 requests, 60,000 tokens in all, 16 heads of 128: 43.8 us, 5.6 TB/s; one of
// 131,072 tokens, 4 heads of 512: 87.3 us, 6.1 TB/s; 32 requests, 4 tokens each, 1,024 seen, 8 heads of 256: 27.5 us, 4.0 TB/s
// (8 us of it start and end: 2.3 us to the first table entry, then every wave's first group at once, 33 MB). A large copy
// moves 4.9 TB/s.
//
// ONCE: one workgroup reads a request's codes of a head, once; they are streamed through the caches (48 requests at head size
// 128 58.8 -> 52.8 us, 131,072 tokens at 512 105.0 -> 93.6; where several workgroups read them, 128 vectors over 32,768
// tokens, 80 -> 88). The rule goes by one request's query vectors alone: it does not see that requests whose tables share
// blocks read the same codes (one token each of 16 branches over a prompt of 8,192 tokens, 16 heads of 128, takes 59 us, of 16
// requests with blocks of their own 90; without the streaming not measured).
template <int D, int NT, bool ONCE>
__global__ __launch_bounds__(kAttendThreads, attend_waves(D, NT)) void attend_kernel(
    const AttendParams p) {
  constexpr int kLoads = D / 32;       // KiB of keys, and of values, in a group
  constexpr int kChunks = D / 64;      // 64-element chunks of a key tile
  constexpr int kSlab = slab_of(D, NT);
  constexpr int kVectors = 16 * NT;
  __shared__ int s_part[kAttendWaves][1];
  __shared__ Seen s_seen;
  __shared__ int s_at[2];
  __shared__ float s_m[kAttendWaves][kVectors], s_l[kAttendWaves][kVectors];
  // (arrays of their own: a read then waits for the copies into its own array and no others)
  __shared__ __align__(16) char s_keys[ring_bytes(D) > sums_bytes(D, NT) ? ring_bytes(D) : sums_bytes(D, NT)];
  __shared__ __align__(16) char s_values[ring_bytes(D)];
  __shared__ u32x4 s_q[kVectors * D / 8];
  float(*const s_o)[kVectors][kSlab + 4] = reinterpret_cast<float(*)[kVectors][kSlab + 4]>(s_keys);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, quad = lane >> 4;
  KA_LDS char* const key_ring = (KA_LDS char*)s_keys + wave * (kCacheGroup * D);
  KA_LDS char* const value_ring = (KA_LDS char*)s_values + wave * (kCacheGroup * D);
  const int heads = p.c.kv_heads, b = p.c.block_log2;
  const int h = blockIdx.y % heads, vector0 = (blockIdx.y / heads) * kVectors;

  // a chunk of requests, one a thread: their units, summed up to each and over all of them
  Seen own;
  int v[1], all[1];
  auto scan = [&](int c0) {
    own = Seen{0, 0, 0, 0, 0, 0};
    if (c0 + tid < p.r.n_seq) own = seen_of(p, c0 + tid);
    v[0] = weight_of(own.units);
    block_scan<kAttendThreads, 1>(v, all, s_part);
  };
  int total = 0, c0 = 0, c_end = p.r.n_seq, u0, u1;
  if (p.whole) {  // workgroup i takes request i
    c0 = blockIdx.x;
    c_end = c0 + 1;
    own = seen_of(p, c0);
    all[0] = total = own.units;
    v[0] = 0;
    if (tid != 0) own.units = 0;  // (thread 0's)
    u0 = 0;
    u1 = total;
  } else {
    for (int c = 0; c < p.r.n_seq; c += kAttendThreads) {
      if (c > 0) __syncthreads();
      scan(c);
      total += all[0];
    }
    total = max(total - kStart, 0);  // (none comes after the last)
    const Shares shares(total, p.parts);
    u0 = min(shares.begin(blockIdx.x), total);  // (workgroups past the shares: none)
    u1 = min(shares.begin(blockIdx.x + 1), total);
  }
  const bool writes_units = !p.whole && blockIdx.x == 0 && blockIdx.y == 0;
  if (writes_units && tid == 0) p.units[p.r.n_seq] = total;
  if (u0 >= u1) return;

  int carry = 0;
  for (; c0 < c_end && (writes_units || carry < u1); c0 += kAttendThreads) {
    if (!p.whole && p.r.n_seq > kAttendThreads) {
      __syncthreads();
      scan(c0);  // (one chunk's sums are there)
    }
    if (writes_units && c0 + tid < p.r.n_seq) p.units[c0 + tid] = carry + v[0];
    const int to = min(u1, carry + all[0] - (p.whole ? 0 : kStart));  // (what the last request counts more has none behind it)
    for (int at = max(u0, carry); at < to;) {
      // the request that `at` lies in, or the one behind the gap that it lies in: one thread's
      const int unit = at - carry - v[0];
      if (own.units > 0 && unit < own.units && unit >= (v[0] > 0 ? -kStart : 0)) {
        s_seen = own;
        s_at[0] = tid;
        s_at[1] = v[0];
      }
      lds_barrier();
      const Seen s = {uniform(s_seen.tokens), uniform(s_seen.row),   uniform(s_seen.queries),
                      uniform(s_seen.first),  uniform(s_seen.groups), uniform(s_seen.units)};
      const int i = c0 + uniform(s_at[0]);
      const int begin = carry + uniform(s_at[1]), end = begin + s.units;
      at = max(at, begin);
      if (at >= to) break;
      const int stop = min(to, end);
      const int g0 = s.first + at - begin;
      const int g1 = s.groups > 0 ? s.first + stop - begin : g0;
      at = stop;
      const int vectors = (int)min<int64_t>((int64_t)min(s.queries, p.max_q) * p.group - vector0, kVectors);
      if (vectors <= 0) {
        lds_barrier();  // s_seen is read
        continue;
      }

      // the query vectors' operands (entry (2 c + k) * NT + n, one lane's 16 bytes after the other), and the keys that each
      // vector sees: lo .. hi
      constexpr int kMine = (2 * kChunks + kAttendWaves - 1) / kAttendWaves;  // of the entries of a tile, this wave's
      u32x4 q_mine[NT][kMine];
      int lo[NT], hi[NT];
      const int shift = s.tokens - s.queries;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int vec = vector0 + 16 * n + col;
        const bool valid = 16 * n + col < vectors;
        const int pos = valid ? position_of(vec, p) : 0;
        const uint16_t* const src =
            p.q + (s.row + (int64_t)pos) * p.sq_t + (int64_t)(h * p.group + (valid ? vec - pos * p.group : 0)) * p.sq_h;
#pragma unroll
        for (int c = 0; c < kMine; ++c) {
          const int e = wave + c * kAttendWaves;
          if (2 * kChunks >= kAttendWaves || e < 2 * kChunks)
            q_mine[n][c] = *reinterpret_cast<const u32x4*>(src + (e >> 1) * 64 + quad * 16 + (e & 1) * 8);
        }
        lo[n] = p.left < 0 ? 0 : pos + shift - p.left;
        hi[n] = p.right < 0 ? s.tokens - 1 : (int)min<int64_t>((int64_t)pos + shift + p.right, s.tokens - 1);
      }
      // groups that every vector sees whole
      const int pos_first = position_of(vector0, p), pos_last = position_of(vector0 + vectors - 1, p);
      const int full_lo = p.left < 0 ? 0 : pos_last + shift - p.left;
      const int full_hi =
          p.right < 0 ? s.tokens - 1 : (int)min<int64_t>((int64_t)pos_first + shift + p.right, s.tokens - 1);

      f32x4 o[NT][D / 16];
      float top[NT], sum[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        top[n] = -INFINITY;
        sum[n] = 0.f;
#pragma unroll
        for (int t = 0; t < D / 16; ++t) o[n][t] = f32x4{0.f, 0.f, 0.f, 0.f};
      }

      const int32_t* const table = p.r.table + (int64_t)i * p.r.table_stride;
      const int lane_offset = col * 64 + quad * 16;
      int ids = 0;
      float k_scales = 1.f, v_scales = 1.f;
      // lane k looks up the wave's groups g + 4 k
      auto look_up = [&](int g) {
        const int mine = min(g + lane * kAttendWaves, g1 - 1);
        ids = table[mine >> (b - 5)];
        if (ids < 0 || ids >= p.c.blocks) ids = -1;
        const float2 sc = *reinterpret_cast<const float2*>(p.c.scales + 2 * ((int64_t)max(ids, 0) * heads + h));
        k_scales = ids < 0 ? 1.f : sc.x;  // (zeros under another block's scale, NaN where it was never written, could be NaN)
        v_scales = ids < 0 ? 1.f : sc.y;
      };
      // One group's codes into the wave's ring, 16 bytes a lane and KiB; zeros for a block that is not of the pool, and where
      // there is no group (so that every turn of the loop issues the same copies, and a wait can count them).
      auto copy = [&](const uint8_t* from, KA_LDS char* to, int g, int k, bool any) {
        const int id = __builtin_amdgcn_readlane(ids, k & 63);
        const int64_t head = (int64_t)max(id, 0) * heads + h;
        const uint8_t* const src = from + ((head << b) + (int64_t)(g & ((1 << (b - 5)) - 1)) * kCacheGroup) * D;
        const __amdgpu_buffer_rsrc_t r =
            __builtin_amdgcn_make_buffer_rsrc((void*)src, (short)0, any && id >= 0 ? kCacheGroup * D : 0, kBufferFlags);
#pragma unroll
        for (int t = 0; t < kLoads; ++t)
          __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (KA_LDS void*)(to + t * 1024), 16, lane_offset, t * 1024, 0,
                                                   ONCE ? kCopyStream : 0);
      };
      auto tile = [&](const KA_LDS char* ring, int t) {
        return *reinterpret_cast<const KA_LDS u32x4*>(ring + t * 1024 + lane * 16);
      };
      // all but the last issued group's keys, or values, have arrived / the reads of the ring are done
      auto arrived = [&]() {
        wait_vmcnt<kLoads>();
        asm volatile("" ::: "memory");
      };
      auto read_out = [&]() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); };

      int k = 0;
      const bool some = g0 + wave < g1;
      if (some) look_up(g0 + wave);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < kMine; ++c) {
          const int e = wave + c * kAttendWaves;
          if (2 * kChunks >= kAttendWaves || e < 2 * kChunks) s_q[(e * NT + n) * 64 + lane] = q_mine[n][c] ^ p.sign;
        }
      if (some) {
        copy(p.c.keys, key_ring, g0 + wave, 0, true);
        copy(p.c.values, value_ring, g0 + wave, 0, true);
      }
      lds_barrier();
      for (int g = g0 + wave; g < g1; g += kAttendWaves) {
        const float k_scale = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(k_scales), k));
        const float v_scale = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v_scales), k));
        const int next = g + kAttendWaves;
        arrived();
        f32x4 st[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) st[n][0] = st[n][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 2 * kChunks; ++c) {
          bf16x8 q[NT];
#pragma unroll
          for (int n = 0; n < NT; ++n) q[n] = __builtin_bit_cast(bf16x8, s_q[(c * NT + n) * 64 + lane]);
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const u32x4 w = tile(key_ring, t * kChunks + (c >> 1));
            const bf16x8 a = operand(w[2 * (c & 1)], w[2 * (c & 1) + 1], k_scale);
#pragma unroll
            for (int n = 0; n < NT; ++n) st[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, q[n], st[n][t], 0, 0, 0);
          }
        }
        read_out();
        if (++k == 64 && next < g1) {
          look_up(next);
          k = 0;
        }
        copy(p.c.keys, key_ring, next, k, next < g1);

        const int key0 = g * kCacheGroup;
        const bool masked = key0 < full_lo || key0 + kCacheGroup - 1 > full_hi;
        bf16x8 weight[NT][2];
        unsigned is_seen[NT];  // one bit of each of the lane's eight keys
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = st[n][e >> 2][e & 3];
          is_seen[n] = 0;
          if (masked) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int key = key0 + (e >> 2) * 16 + quad * 4 + (e & 3);
              const bool sees = key >= lo[n] && key <= hi[n];
              x[e] = sees ? x[e] : -INFINITY;
              is_seen[n] |= sees ? 1u << e : 0u;
            }
          }
          float best = max3(max3(x[0], x[1], x[2]), max3(x[3], x[4], x[5]), max3(x[6], x[7], x[7]));
          best = column_max(best) * p.scale;
          // the running maximum is raised (and O rescaled) only where it grows by more than 2^8: weights are then at most 2^8
          if (__any(!(best <= top[n] + 8.f) && best != -INFINITY)) {
            const float up = __builtin_elementwise_maximum(top[n], best);
            const float f = top[n] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top[n] - up);
            top[n] = up;
            sum[n] *= f;
#pragma unroll
            for (int t = 0; t < D / 16; ++t) o[n][t] *= f;
          }
          const float base = top[n] == -INFINITY ? 0.f : top[n];
          float w[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], p.scale, -base));
          u32x4 high, low;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            high[e] = pair_of(w[2 * e], w[2 * e + 1]);
            low[e] = pair_of(w[2 * e] - __uint_as_float(high[e] << 16),
                             w[2 * e + 1] - __uint_as_float(high[e] & 0xffff0000u));
          }
          weight[n][0] = __builtin_bit_cast(bf16x8, high);
          weight[n][1] = __builtin_bit_cast(bf16x8, low);
          const float add = ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
          sum[n] += add;
        }

        arrived();
        bool nan = false;
        if (masked) {
          unsigned any = 0;
#pragma unroll
          for (int t = 0; t < kLoads; ++t) {
            const u32x4 w = tile(value_ring, t);
#pragma unroll
            for (int e = 0; e < 4; ++e) any |= nan_codes(w[e]);
          }
          nan = __any(any != 0);
        }
        if (nan) {  // a NaN reaches the vectors that see its token, and no others (zero times NaN would be NaN)
#pragma unroll
          for (int t = 0; t < kLoads; ++t) {
            u32x4 w = tile(value_ring, t);
            u32x4 f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              f[e] = nan_codes(w[e]);
              w[e] &= ~((f[e] >> 7) * 255u);
            }
#pragma unroll
            for (int d = 0; d < 2; ++d) {
              const bf16x8 marks = operand(f[2 * d] >> 1, f[2 * d + 1] >> 1, 1.f);  // 2.0 where NaN
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                bf16x8 sees;
#pragma unroll
                for (int e = 0; e < 8; ++e) sees[e] = is_seen[n] >> e & 1 ? (__bf16)1.f : (__bf16)0.f;
                const f32x4 count =
                    __builtin_amdgcn_mfma_f32_16x16x32_bf16(marks, sees, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[n][2 * t + d][e] += count[e] > 0.f ? NAN : 0.f;
              }
            }
            *reinterpret_cast<KA_LDS u32x4*>(value_ring + t * 1024 + lane * 16) = w;
          }
        }
#pragma unroll
        for (int t = 0; t < kLoads; ++t) {
          const u32x4 w = tile(value_ring, t);
#pragma unroll
          for (int d = 0; d < 2; ++d) {
            const bf16x8 a = operand(w[2 * d], w[2 * d + 1], v_scale);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              o[n][2 * t + d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, weight[n][0], o[n][2 * t + d], 0, 0, 0);
              o[n][2 * t + d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, weight[n][1], o[n][2 * t + d], 0, 0, 0);
            }
          }
        }
        read_out();
        copy(p.c.values, value_ring, next, k, next < g1);
      }

      wait_vmcnt<0>();  // (the copies of no group, into what the sums take)

      // join the waves
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float l = column_sum(sum[n]);
        if (quad == 0) {
          s_m[wave][16 * n + col] = top[n];
          s_l[wave][16 * n + col] = l;
        }
      }
      lds_barrier();
      // vector c's maximum and sum over the waves
      auto top_of = [&](int c) {
        float up = s_m[0][c];
#pragma unroll
        for (int w = 1; w < kAttendWaves; ++w) up = __builtin_elementwise_maximum(up, s_m[w][c]);
        return up;
      };
      auto total_of = [&](int c, float up) {
        float l = 0.f;
#pragma unroll
        for (int w = 0; w < kAttendWaves; ++w)
          l += s_m[w][c] == -INFINITY ? 0.f : s_l[w][c] * __builtin_amdgcn_exp2f(s_m[w][c] - up);
        return l;
      };
      const bool whole = begin >= u0 && end <= u1;
      float* const part =
          p.partial + (((int64_t)blockIdx.y * p.parts + blockIdx.x) * 2 + (begin <= u0 ? 0 : 1)) * (kVectors * (D + 2));
      if (!whole && tid < vectors) {
        const float up = top_of(tid);
        part[kVectors * D + tid] = up;
        part[kVectors * D + kVectors + tid] = total_of(tid, up);
      }
      for (int d0 = 0; d0 < D; d0 += kSlab) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float f = top[n] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top[n] - top_of(16 * n + col));
#pragma unroll
          for (int t = 0; t < D / 16; ++t)
            if (t * 16 >= d0 && t * 16 < d0 + kSlab)
              *reinterpret_cast<f32x4*>(&s_o[wave][16 * n + col][t * 16 - d0 + quad * 4]) = o[n][t] * f;
        }
        lds_barrier();
        for (int e = tid; e < vectors * (kSlab / 4); e += kAttendThreads) {
          const int c = e / (kSlab / 4), d = (e % (kSlab / 4)) * 4;
          f32x4 x = *reinterpret_cast<const f32x4*>(&s_o[0][c][d]);
#pragma unroll
          for (int w = 1; w < kAttendWaves; ++w) x += *reinterpret_cast<const f32x4*>(&s_o[w][c][d]);
          if (whole) {
            const float l = total_of(c, top_of(c));
            const int vec = vector0 + c, pos = position_of(vec, p), head = h * p.group + vec - pos * p.group;
            if (l == 0.f) x = f32x4{0.f, 0.f, 0.f, 0.f}; else x = x * (1.f / l);
            *reinterpret_cast<u32x2*>(p.o + (s.row + (int64_t)pos) * p.so_t + head * p.so_h + d0 + d) =
                u32x2{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])};
          } else {
            *reinterpret_cast<f32x4*>(part + c * D + d0 + d) = x;
          }
        }
        lds_barrier();
      }
    }
    carry += all[0];
  }
  if (p.whole) fill_past<D>(p, seen_of(p, blockIdx.x), blockIdx.y, tid, kAttendThreads);
}

// Joins a request's shares: O = sum of 2^(m_w - M) O_w over sum of 2^(m_w - M) l_w, in an order that the sizes alone set.
// Requests that one workgroup took whole are done already. Up to kFew shares: a thread walks them for four elements of a
// vector. More: 64 elements of a vector by 16 threads of four and 16 rows, each row with every sixteenth share (so that
// up to 16 cost one round of loads), and the rows joined through LDS. 4.4 to 6.6 us, launch and four rounds of loads; 33 us with
// one walk over 64 shares of one request.
template <int D>
__global__ __launch_bounds__(256) void join_kernel(const AttendParams p, int vectors_per) {
  constexpr int kSlabs = D / 64, kFew = 4;
  __shared__ float s_m[16], s_l[16];
  __shared__ f32x4 s_x[16][16];
  const int i = blockIdx.x, heads = p.c.kv_heads;
  const int total = p.units[p.r.n_seq], begin = p.units[i];
  const Seen s = seen_of(p, i);
  if (s.units == 0) return;
  fill_past<D>(p, s, blockIdx.y, blockIdx.z * 256 + threadIdx.x, gridDim.z * 256);
  const Shares shares(total, p.parts);
  const int first = shares.part_of(begin), last = shares.part_of(begin + s.units - 1);
  if (first == last) return;
  const int h = blockIdx.y % heads, vector0 = (blockIdx.y / heads) * vectors_per;
  const int vectors = (int)min<int64_t>((int64_t)min(s.queries, p.max_q) * p.group - vector0, vectors_per);
  const int64_t size = (int64_t)vectors_per * (D + 2);
  const float* const base = p.partial + (int64_t)blockIdx.y * p.parts * 2 * size;
  const int tid = threadIdx.x;

  struct Sum {
    float up, l;
    f32x4 x;
  };
  auto add = [&](Sum& a, int w, int c, int d) {
    // (only the first share can have begun before the request: then the request is its workgroup's second)
    const float* const part = base + (2 * (int64_t)w + (w == first && begin > shares.begin(w) ? 1 : 0)) * size;
    const float m = part[vectors_per * D + c], lw = part[vectors_per * D + vectors_per + c];
    const f32x4 xw = *reinterpret_cast<const f32x4*>(part + c * D + d);
    const float next = __builtin_elementwise_maximum(a.up, m);
    const float fo = a.up == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(a.up - next);
    const float fw = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - next);
    a.x = a.x * fo + xw * fw;
    a.l = a.l * fo + lw * fw;
    a.up = next;
  };
  auto store = [&](const Sum& a, int c, int d) {
    const int vec = vector0 + c, pos = position_of(vec, p), head = h * p.group + vec - pos * p.group;
    const f32x4 x = a.l == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : a.x * (1.f / a.l);
    *reinterpret_cast<u32x2*>(p.o + (s.row + (int64_t)pos) * p.so_t + head * p.so_h + d) =
        u32x2{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])};
  };
  const Sum none = {-INFINITY, 0.f, f32x4{0.f, 0.f, 0.f, 0.f}};
  if (last - first < kFew) {
    for (int e = blockIdx.z * 256 + tid; e < vectors * (D / 4); e += gridDim.z * 256) {
      const int c = e / (D / 4), d = (e % (D / 4)) * 4;
      Sum a = none;
#pragma unroll
      for (int w = 0; w < kFew; ++w)
        if (first + w <= last) add(a, first + w, c, d);
      store(a, c, d);
    }
    return;
  }
  const int row = tid >> 4, lane = tid & 15;
  for (int e = blockIdx.z; e < vectors * kSlabs; e += gridDim.z) {
    const int c = e / kSlabs, d = (e % kSlabs) * 64 + lane * 4;
    Sum a = none;
#pragma unroll 2
    for (int w = first + row; w <= last; w += 16) add(a, w, c, d);
    __syncthreads();  // the last round's sums are read
    s_x[row][lane] = a.x;
    if (lane == 0) {
      s_m[row] = a.up;
      s_l[row] = a.l;
    }
    __syncthreads();
    if (row == 0) {
      a = none;
#pragma unroll
      for (int w = 0; w < 16; ++w) a.up = __builtin_elementwise_maximum(a.up, s_m[w]);
#pragma unroll
      for (int w = 0; w < 16; ++w) {
        const float f = s_m[w] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s_m[w] - a.up);
        a.x += s_x[w][lane] * f;
        a.l += s_l[w] * f;
      }
      store(a, c, d);
    }
  }
}

template <int D, int NT>
void launch(const AttendParams& p, const AttendShape& s, hipStream_t stream) {
  const unsigned y = (unsigned)(p.c.kv_heads * s.tiles), x = (unsigned)(p.whole ? p.r.n_seq : s.parts);
  if (s.tiles == 1)
    attend_kernel<D, NT, true><<<dim3(x, y), dim3(kAttendThreads), 0, stream>>>(p);
  else
    attend_kernel<D, NT, false><<<dim3(x, y), dim3(kAttendThreads), 0, stream>>>(p);
  if (p.whole) return;
  // a workgroup for 64 elements of each vector, or as many as fill the GPU several times over
  const int64_t pairs = (int64_t)p.r.n_seq * y, most = (2048 + pairs - 1) / pairs, items = (int64_t)s.used * (D / 64);
  const unsigned z = (unsigned)(items < most ? items : most);
  join_kernel<D><<<dim3((unsigned)p.r.n_seq, y, z), dim3(256), 0, stream>>>(p, 16 * NT);
}

}  // namespace

AttendShape attend_shape(const CacheRef& c, int32_t n_seq, int32_t group, int32_t max_q, int64_t seen) {
  AttendShape s;
  const int64_t vectors = (int64_t)max_q * group;
  const int most = c.head_dim <= 128 ? 4 : c.head_dim == 256 ? 2 : 1;  // tiles of 16 vectors that the registers hold
  const int tiles = vectors <= 16 || most == 1 ? 1 : vectors <= 32 || most == 2 ? 2 : 4;
  s.vectors = 16 * tiles;
  s.tiles = (int)((vectors + s.vectors - 1) / s.vectors);
  if (s.tiles < 1) s.tiles = 1;
  const int at_once = attend_waves(c.head_dim, tiles);
  const int64_t y = (int64_t)c.kv_heads * s.tiles;
  const int64_t parts = 256 * at_once / y;
  s.parts = parts < 1 ? 1 : (int)parts;
  s.used = (int)(vectors < s.vectors ? vectors : s.vectors);
  s.whole = seen <= (c.head_dim == 512 ? kWholeTokens / 4 : kWholeTokens);
  s.units_bytes = (4 * ((int64_t)n_seq + 1) + 255) / 256 * 256;
  s.bytes = s.whole ? 0 : s.units_bytes + y * s.parts * 2 * s.vectors * (c.head_dim + 2) * 4;
  return s;
}

hipError_t launch_cache_attend(const AttendParams& p, const AttendShape& s, hipStream_t stream) {
  switch (p.c.head_dim * 8 + s.vectors / 16) {
    case 64 * 8 + 1: launch<64, 1>(p, s, stream); break;
    case 64 * 8 + 2: launch<64, 2>(p, s, stream); break;
    case 64 * 8 + 4: launch<64, 4>(p, s, stream); break;
    case 128 * 8 + 1: launch<128, 1>(p, s, stream); break;
    case 128 * 8 + 2: launch<128, 2>(p, s, stream); break;
    case 128 * 8 + 4: launch<128, 4>(p, s, stream); break;
    case 256 * 8 + 1: launch<256, 1>(p, s, stream); break;
    case 256 * 8 + 2: launch<256, 2>(p, s, stream); break;
    case 512 * 8 + 1: launch<512, 1>(p, s, stream); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace karpo
