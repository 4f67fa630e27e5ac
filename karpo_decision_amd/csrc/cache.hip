// The block cache (karpo_cache.h): reserving blocks, appending keys and values in 8 bits, reading them back.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "cache.h"
#include "cache_common.h"
#include "karpo_cache.h"

namespace karpo {

namespace {

// ---- reserve

constexpr int kReserveThreads = 1024;

struct Request {
  int tokens, count, held, need, touched;  // held, need: blocks; touched: blocks that get tokens
};

// One launch: every workgroup adds up all requests by itself (a few hundred loads that L2 holds) and then writes the rows
// of its own range, so nothing waits on another workgroup. A new block's first token, and a request's first new token, write
// the block's entries; which block a token's is follows from the sums alone. Bound by the launch and one round of dependent
// loads at a decoding step's size, by the 12 bytes a row it stores at a prompt's.
__global__ __launch_bounds__(kReserveThreads) void reserve_kernel(const ReserveParams p) {
  __shared__ int s_first[kReserveThreads + 1], s_need[kReserveThreads], s_write[kReserveThreads],
      s_tokens[kReserveThreads];
  __shared__ int s_part[kReserveThreads / 64][4];
  const int tid = threadIdx.x;
  const int b = p.block_log2, block = 1 << b;

  const int free_count = *p.free_count;
  const bool bad_list = free_count < 0 || free_count > p.free_capacity;
  // request i and whether it is out of range (then it counts as none)
  auto take = [&](int i, bool* bad) {
    Request r = {0, 0, 0, 0, 0};
    if (i >= p.n_seq) return r;
    r.tokens = p.lengths[i];
    r.count = p.counts[i];
    if (r.tokens < 0 || r.count < 0 || (int64_t)r.tokens + r.count > p.most || r.count > p.rows) {
      *bad = true;
      r.tokens = r.count = 0;
    }
    const int after = r.tokens + r.count, round = block - 1;
    r.held = (r.tokens + round) >> b;
    r.need = ((after + round) >> b) - r.held;
    r.touched = r.count > 0 ? ((after - 1) >> b) - (r.tokens >> b) + 1 : 0;
    return r;
  };
  // Of a chunk of requests: the sums before each (rows, blocks taken, blocks written) and over all of them. The fourth, of
  // counts / 2,048, tells a sum of rows that 32 bits do not hold: where it is within `rows` / 2,048, they do.
  Request r;
  bool bad = bad_list;
  int v[4], all[4];
  auto scan = [&](int c0) {
    r = take(c0 + tid, &bad);
    v[0] = r.count;
    v[1] = r.need;
    v[2] = r.touched;
    v[3] = r.count >> 11;
    block_scan<kReserveThreads, 4>(v, all, s_part);
  };
  int64_t total = 0, need = 0;
  for (int c0 = 0; c0 < p.n_seq; c0 += kReserveThreads) {
    if (c0 > 0) __syncthreads();
    scan(c0);
    total += all[3] > p.rows >> 11 ? (int64_t)p.rows + 1 : (int64_t)(unsigned)all[0];
    need += all[1];
  }
  bad = __syncthreads_or(bad);
  const int status = bad || total > p.rows ? KARPO_CACHE_BAD_LENGTHS : need > free_count ? KARPO_CACHE_NO_BLOCKS : 0;

  const int r0 = (int)ka_min64((int64_t)blockIdx.x * p.per, p.rows);
  const int r1 = (int)ka_min64((int64_t)r0 + p.per, p.rows);
  int carry[3] = {0, 0, 0};  // rows, blocks taken, writes before the chunk's requests
  for (int c0 = 0; c0 < p.n_seq; c0 += kReserveThreads) {
    const int i = c0 + tid, m = min(kReserveThreads, p.n_seq - c0);
    if (p.n_seq > kReserveThreads) scan(c0);  // (one chunk's sums are there)
    if (status != 0) r.count = v[0] = v[1] = v[2] = all[0] = all[1] = all[2] = 0;
    if (tid < m) {
      s_first[tid] = carry[0] + v[0];
      s_need[tid] = carry[1] + v[1];
      s_write[tid] = carry[2] + v[2];
      s_tokens[tid] = r.tokens;
    }
    if (tid == 0) s_first[m] = carry[0] + all[0];
    if (blockIdx.x == 0 && i < p.n_seq) {
      p.q_cu[i] = carry[0] + v[0];
      p.new_lengths[i] = status == 0 ? r.tokens + r.count : p.lengths[i];
    }
    __syncthreads();
    const int hi = min(r1, s_first[m]);
    for (int row = max(r0, s_first[0]) + tid; row < hi; row += kReserveThreads) {
      const int j = last_at_most(s_first, m, row);
      const int first = s_first[j], tokens = s_tokens[j];
      const int position = tokens + row - first;
      const int at = position >> b, inside = position & (block - 1);
      const int held = (tokens + block - 1) >> b;
      const bool fresh = at >= held;
      int32_t* const entry = p.table + (int64_t)(c0 + j) * p.table_stride + at;
      const int id = fresh ? p.free_blocks[free_count - 1 - (s_need[j] + at - held)] : *entry;
      p.slots[row] = ((int64_t)id << b) + inside;
      p.positions[row] = position;
      if (inside == 0 || row == first) {
        if (fresh) *entry = id;
        const int w = s_write[j] + at - (tokens >> b);
        *reinterpret_cast<int4*>(p.writes + 4 * (int64_t)w) =
            make_int4(id, inside, row, min(block - inside, s_first[j + 1] - row));
      }
    }
    for (int k = 0; k < 3; ++k) carry[k] += all[k];
    __syncthreads();  // the next chunk's requests take the arrays
  }
  for (int row = max(r0, carry[0]) + tid; row < r1; row += kReserveThreads) {  // behind the last request
    p.slots[row] = -1;
    p.positions[row] = 0;
  }
  for (int64_t w = carry[2] + (int64_t)blockIdx.x * kReserveThreads + tid; w < p.writes_capacity;
       w += (int64_t)gridDim.x * kReserveThreads)
    *reinterpret_cast<int4*>(p.writes + 4 * w) = make_int4(0, 0, 0, 0);
  if (blockIdx.x == 0 && tid == 0) {
    p.q_cu[p.n_seq] = carry[0];
    *p.free_left = free_count - carry[1];
    *p.status = status;
  }
}

// ---- append

// Four fp32 as e4m3 (nearest, ties to even), past the range at its end, NaN as NaN.
__device__ __forceinline__ float in_range(float x) {
  return x != x ? x : __builtin_amdgcn_fmed3f(x, -448.f, 448.f);
}
__device__ __forceinline__ unsigned codes4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(in_range(a), in_range(b), 0, false);
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(in_range(c), in_range(d), w, true);
}
// Four codes times `f` (a power of two, at most 1), rounded again.
__device__ __forceinline__ unsigned codes_again(unsigned w, float f) {
  const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  return codes4(lo[0] * f, lo[1] * f, hi[0] * f, hi[1] * f);
}

// Largest finite magnitude of packed bf16 pairs, as bits.
__device__ __forceinline__ unsigned largest_of(unsigned best, const u32x4& x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned lo = x[i] & 0x7fffu, hi = (x[i] >> 16) & 0x7fffu;
    best = max(best, lo < 0x7f80u ? lo : 0u);
    best = max(best, hi < 0x7f80u ? hi : 0u);
  }
  return best;
}

// The least e with m <= 448 * 2^e for the bf16 magnitude with these bits (448 = 1.75 * 2^8).
__device__ __forceinline__ int exponent_of(unsigned bits) {
  const int e = (int)(bits >> 7) - 127 - 8 + ((bits & 0x7f) > 0x60 ? 1 : 0);
  return min(max(e, KARPO_CACHE_MIN_EXP), KARPO_CACHE_MAX_EXP);
}

// One write's keys, or values, of one head: WAVES waves, each of TILES KiB of codes, all rows in registers between the
// maximum and the rounding. A key tile's lane takes 16 elements of one token (two loads, one 16-byte store); a value tile's
// takes 8 tokens x 16 elements, the tokens that lie side by side in the cache, so both sides move 16 bytes a lane and
// nothing goes through LDS. Tokens beside the write keep their bytes: where a 16-byte piece holds some, it is read and
// merged (the block is this workgroup's alone).
template <int TILES, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void append_kernel(const AppendParams p) {
  const int heads = p.c.kv_heads;
  const int64_t unit = blockIdx.x / (2 * heads);
  const int which = (int)(blockIdx.x - unit * 2 * heads), h = which >> 1;
  const bool value = which & 1;
  const int4 wr = *reinterpret_cast<const int4*>(p.writes + 4 * unit);
  const int id = wr.x, first = wr.y, row = wr.z, count = wr.w;
  const int block = 1 << p.c.block_log2, d = p.c.head_dim;
  if (count < 1 || id < 0 || id >= p.c.blocks || first < 0 || count > block - first || row < 0 || row > p.rows - count)
    return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t head = (int64_t)id * heads + h;
  uint8_t* const out = (value ? p.c.values : p.c.keys) + (head << p.c.block_log2) * d;
  const int64_t stride = value ? p.sv_t : p.sk_t;
  const uint16_t* const in = (value ? p.v + h * p.sv_h : p.k + h * p.sk_h) + ((int64_t)row - first) * stride;

  // keys: tile i of the wave, token lane / 4 of its 16, elements (lane % 4) * 16 of its 64: x[2 i], x[2 i + 1]
  const int k_chunks = d >> 6;
  // values: lanes 8 i .. 8 i + 7 take tile i of the wave's 8; q = lane % 4, the tokens 16 t + 4 q + i as x[2 (4 t + i)] at
  // elements 8 * (lane / 4 % 2) .. + 8 and x[2 (4 t + i) + 1] 16 further on
  const int v_tile = wave * TILES + (lane >> 3), v_chunks = d >> 5;
  const int v_token = (v_tile / v_chunks) * 32 + (lane & 3) * 4, v_elem = (v_tile % v_chunks) * 32 + ((lane >> 2) & 1) * 8;
  const bool v_lane = (lane >> 3) < TILES;
  const u32x4 zero = {0, 0, 0, 0};
  u32x4 x[16];
  unsigned best = 0;
  if (!value) {
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
      const int tile = wave * TILES + i, token = (tile / k_chunks) * 16 + (lane >> 2);
      const uint16_t* const src = in + token * stride + (tile % k_chunks) * 64 + (lane & 3) * 16;
      const bool mine = token >= first && token < first + count;
      x[2 * i] = mine ? *reinterpret_cast<const u32x4*>(src) : zero;
      x[2 * i + 1] = mine ? *reinterpret_cast<const u32x4*>(src + 8) : zero;
    }
#pragma unroll
    for (int i = 0; i < TILES * 2; ++i) best = largest_of(best, x[i]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int token = v_token + (j >> 2) * 16 + (j & 3);
      const uint16_t* const src = in + token * stride + v_elem;
      const bool mine = v_lane && token >= first && token < first + count;
      x[2 * j] = mine ? *reinterpret_cast<const u32x4*>(src) : zero;
      x[2 * j + 1] = mine ? *reinterpret_cast<const u32x4*>(src + 16) : zero;
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) best = largest_of(best, x[j]);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) best = max(best, (unsigned)__shfl_xor((int)best, o));
  if constexpr (WAVES > 1) {
    __shared__ unsigned s_best[WAVES];
    if (lane == 0) s_best[wave] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) best = max(best, s_best[w]);
  }
  int e = exponent_of(best);
  float again = 1.f;  // what the earlier tokens' codes are multiplied by
  float* const scale = p.c.scales + 2 * head + (value ? 1 : 0);
  if (first > 0) {
    const int old = min(max((int)((__float_as_uint(*scale) >> 23) & 0xff) - 127, KARPO_CACHE_MIN_EXP), KARPO_CACHE_MAX_EXP);
    e = max(e, old);
    again = power_of_two(max(old - e, -126));  // (448 * 2^-126 rounds to zero too)
  }
  const bool grown = again != 1.f;
  const float inv = power_of_two(-e);
  if constexpr (WAVES > 1) __syncthreads();  // every wave has read the old scale
  if (threadIdx.x == 0) *scale = power_of_two(e);

  if (!value) {
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
      const int tile = wave * TILES + i, token = (tile / k_chunks) * 16 + (lane >> 2);
      u32x4* const dst = reinterpret_cast<u32x4*>(out + tile * 1024 + lane * 16);
      u32x4 w;
      if (token >= first && token < first + count) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const u32x4& s = x[2 * i + (j >> 1)];
          const int o = (j & 1) * 4;
          w[j] = codes4(bf16_at(s, o) * inv, bf16_at(s, o + 1) * inv, bf16_at(s, o + 2) * inv, bf16_at(s, o + 3) * inv);
        }
        *dst = w;
      } else if (grown && token < first) {
        w = *dst;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = codes_again(w[j], again);
        *dst = w;
      }
    }
    return;
  }
  // bytes of the tokens 16 t + 4 q + 0 .. 3 that are new, and that are rounded again
  unsigned is_new[2] = {0, 0}, is_old[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int token = v_token + (j >> 2) * 16 + (j & 3);
    const unsigned byte = 0xffu << (8 * (j & 3));
    if (token >= first && token < first + count) is_new[j >> 2] |= byte;
    if (grown && token < first) is_old[j >> 2] |= byte;
  }
  if (!v_lane || (is_new[0] | is_new[1] | is_old[0] | is_old[1]) == 0) return;
  const bool whole = (is_new[0] & is_new[1]) == 0xffffffffu;
  u32x4* const dst = reinterpret_cast<u32x4*>(out + v_tile * 1024 + ((lane >> 2) & 1) * 512 + (lane & 3) * 16);
#pragma unroll
  for (int s = 0; s < 8; ++s) {
    u32x4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // dh = j / 2, t = j % 2
      const int t = j & 1, dh = j >> 1;
      w[j] = codes4(bf16_at(x[2 * (4 * t) + dh], s) * inv, bf16_at(x[2 * (4 * t + 1) + dh], s) * inv,
                    bf16_at(x[2 * (4 * t + 2) + dh], s) * inv, bf16_at(x[2 * (4 * t + 3) + dh], s) * inv);
    }
    if (!whole) {
      const u32x4 was = dst[4 * s];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned n = is_new[j & 1], o = is_old[j & 1];
        const unsigned old = o != 0 ? (codes_again(was[j], again) & o) | (was[j] & ~o) : was[j];
        w[j] = (w[j] & n) | (old & ~n);
      }
    }
    dst[4 * s] = w;
  }
}

// ---- read

constexpr int kReadWaves = 4;

// 32 tokens of one head, keys or values, per wave and turn. A key tile's lane turns 16 codes into 32 bytes of one row; a
// value tile's holds 8 tokens x 8 elements (four 16-byte loads), which it turns into four elements of each token's row
// twice. Each workgroup adds up all lengths by itself and takes an equal share of all groups of 32 tokens.
__global__ __launch_bounds__(64 * kReadWaves) void read_kernel(const ReadParams p) {
  constexpr int kThreads = 64 * kReadWaves;
  __shared__ int s_group[kThreads + 1], s_row[kThreads], s_start[kThreads], s_tokens[kThreads];
  __shared__ int s_part[kReadWaves][2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int h = blockIdx.y >> 1, heads = p.c.kv_heads, d = p.c.head_dim, b = p.c.block_log2;
  const bool value = blockIdx.y & 1;

  // first and last token of request i that are read
  auto range = [&](int i, int* start, int* tokens) {
    *tokens = min(max(p.r.lengths[i], 0), p.r.most);
    *start = 0;
    if (p.q_cu != nullptr) {
      const int queries = p.q_cu[i + 1] - p.q_cu[i];
      if (queries <= 0) {
        *tokens = 0;
      } else if (p.window_left >= 0) {
        const int64_t s = (int64_t)*tokens - queries - p.window_left;
        *start = s > 0 ? (int)min<int64_t>(s, *tokens) & ~(kCacheGroup - 1) : 0;
      }
    }
  };
  // Of a chunk of requests: groups of 32 rows, and the last group's missing rows, before each and over all.
  int start = 0, tokens = 0, v[2], all[2];
  auto scan = [&](int c0) {
    start = tokens = 0;
    if (c0 + tid < p.r.n_seq) range(c0 + tid, &start, &tokens);
    v[0] = (tokens - start + kCacheGroup - 1) / kCacheGroup;
    v[1] = tokens - start - v[0] * kCacheGroup;
    block_scan<kThreads, 2>(v, all, s_part);
  };
  int64_t groups = 0;
  for (int c0 = 0; c0 < p.r.n_seq; c0 += kThreads) {
    if (c0 > 0) __syncthreads();
    scan(c0);
    groups += all[0];
  }
  const int64_t g0 = groups * blockIdx.x / gridDim.x, g1 = groups * (blockIdx.x + 1) / gridDim.x;

  int64_t carry_groups = 0, carry_rows = 0;
  for (int c0 = 0; c0 < p.r.n_seq; c0 += kThreads) {
    const int i = c0 + tid, m = min(kThreads, p.r.n_seq - c0);
    if (p.r.n_seq > kThreads) {
      __syncthreads();
      scan(c0);  // (one chunk's sums are there)
    }
    const int64_t row = carry_rows + (int64_t)v[0] * kCacheGroup + v[1];
    if (tid < m) {
      s_group[tid] = v[0];
      s_row[tid] = (int)ka_min64(row, INT32_MAX);
      s_start[tid] = start;
      s_tokens[tid] = tokens;
    }
    if (tid == 0) s_group[m] = all[0];
    if (blockIdx.x == 0 && blockIdx.y == 0 && i < p.r.n_seq) p.k_cu[i] = (int)ka_min64(row, INT32_MAX);
    __syncthreads();
    const int64_t hi = ka_min64(g1, carry_groups + all[0]);
    for (int64_t g = (g0 > carry_groups ? g0 : carry_groups) + wave; g < hi; g += kReadWaves) {
      const int u = (int)(g - carry_groups);
      const int j = last_at_most(s_group, m, u);
      const int token0 = s_start[j] + (u - s_group[j]) * kCacheGroup;
      const int64_t out_row = (int64_t)s_row[j] + token0 - s_start[j];
      const int tokens_left = (int)ka_min64(ka_min64(s_tokens[j] - token0, p.rows - out_row), kCacheGroup);
      if (tokens_left <= 0) continue;
      const int id = p.r.table[(int64_t)(c0 + j) * p.r.table_stride + (token0 >> b)];
      const bool known = id >= 0 && id < p.c.blocks;
      const int64_t head = (int64_t)(known ? id : 0) * heads + h;
      const int inside = token0 & ((1 << b) - 1);
      const uint8_t* const src = (value ? p.c.values : p.c.keys) + (head << b) * d + inside * d;
      const float scale = p.c.scales[2 * head + (value ? 1 : 0)];
      uint16_t* const dst = (value ? p.v : p.k) + (out_row * heads + h) * d;
      const int64_t step = (int64_t)heads * d;
      if (!value) {
        const int chunks = d >> 6;
        for (int t = 0; t < 2 * chunks; ++t) {  // tiles of 16 tokens x 64 elements
          const int token = (t / chunks) * 16 + (lane >> 2);
          u32x4 w = *reinterpret_cast<const u32x4*>(src + t * 1024 + lane * 16);
          if (!known) w = u32x4{0, 0, 0, 0};
          if (token >= tokens_left) continue;
          u32x4* const to = reinterpret_cast<u32x4*>(dst + token * step + (t % chunks) * 64 + (lane & 3) * 16);
          to[0] = bf16_of_8(w[0], w[1], scale);
          to[1] = bf16_of_8(w[2], w[3], scale);
        }
      } else {
        const int q = lane & 3, part = (lane >> 2) & 3;
        for (int t = lane >> 4; t < d >> 5; t += 4) {  // tiles of 32 tokens x 32 elements: 16 lanes each
          u32x4 w[4];
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            w[s] = *reinterpret_cast<const u32x4*>(src + t * 1024 + (4 * part + s) * 64 + q * 16);
            if (!known) w[s] = u32x4{0, 0, 0, 0};
          }
#pragma unroll
          for (int dh = 0; dh < 2; ++dh)
#pragma unroll
            for (int j2 = 0; j2 < 4; ++j2) {  // two tokens: 16 (j2 / 2) + 4 q + 2 (j2 % 2) + 0, 1
              const int t2 = j2 >> 1, up = j2 & 1;
              unsigned pair[4];
#pragma unroll
              for (int s = 0; s < 4; ++s) pair[s] = bf16_pair(w[s][2 * dh + t2], scale, up);
              const int token = 16 * t2 + 4 * q + 2 * up;
              uint16_t* const to = dst + token * step + t * 32 + dh * 16 + part * 4;
              if (token < tokens_left)
                *reinterpret_cast<u32x2*>(to) = u32x2{__builtin_amdgcn_perm(pair[1], pair[0], 0x05040100u),
                                                      __builtin_amdgcn_perm(pair[3], pair[2], 0x05040100u)};
              if (token + 1 < tokens_left)
                *reinterpret_cast<u32x2*>(to + step) = u32x2{__builtin_amdgcn_perm(pair[1], pair[0], 0x07060302u),
                                                             __builtin_amdgcn_perm(pair[3], pair[2], 0x07060302u)};
            }
        }
      }
    }
    carry_groups += all[0];
    carry_rows += (int64_t)all[0] * kCacheGroup + all[1];
    __syncthreads();
  }
  if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) p.k_cu[p.r.n_seq] = (int)ka_min64(carry_rows, INT32_MAX);
}

}  // namespace

hipError_t launch_cache_reserve(ReserveParams p, hipStream_t stream) {
  const int64_t most = 512;  // workgroups
  const int64_t groups = ka_min64(most, (p.rows + (int64_t)kReserveThreads - 1) / kReserveThreads);
  const int64_t grid = groups < 1 ? 1 : groups;
  p.per = (int32_t)((p.rows + grid - 1) / grid);
  reserve_kernel<<<dim3((unsigned)grid), dim3(kReserveThreads), 0, stream>>>(p);
  return hipGetLastError();
}

hipError_t launch_cache_append(const AppendParams& p, int64_t n_writes, hipStream_t stream) {
  const dim3 grid((unsigned)(n_writes * 2 * p.c.kv_heads));
  const int tiles = (p.c.head_dim << p.c.block_log2) / 1024;
  switch (tiles) {
    case 2: append_kernel<2, 1><<<grid, dim3(64), 0, stream>>>(p); break;
    case 4: append_kernel<4, 1><<<grid, dim3(64), 0, stream>>>(p); break;
    case 8: append_kernel<8, 1><<<grid, dim3(64), 0, stream>>>(p); break;
    case 16: append_kernel<8, 2><<<grid, dim3(128), 0, stream>>>(p); break;
    case 32: append_kernel<8, 4><<<grid, dim3(256), 0, stream>>>(p); break;
    case 64: append_kernel<8, 8><<<grid, dim3(512), 0, stream>>>(p); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

hipError_t launch_cache_read(const ReadParams& p, hipStream_t stream) {
  // enough workgroups to fill the GPU several times over, no more than the groups of 32 rows ask for
  const int64_t sides = 2 * (int64_t)p.c.kv_heads;
  const int64_t groups = p.rows / kCacheGroup + p.r.n_seq;
  const int64_t wanted = (groups + kReadWaves - 1) / kReadWaves, fill = (256 * 16 + sides - 1) / sides;
  const int64_t x = ka_min64(wanted < 1 ? 1 : wanted, fill);
  read_kernel<<<dim3((unsigned)x, (unsigned)sides), dim3(64 * kReadWaves), 0, stream>>>(p);
  return hipGetLastError();
}

}  // namespace karpo
