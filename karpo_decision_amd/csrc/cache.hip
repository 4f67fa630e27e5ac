// The block cache (karpo_cache.h): reserving blocks, appending keys and values in 8 bits, reading them back.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

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
// the block's entries; which block a token's is follows from the sums alone. Bound by the launch and three rounds of dependent
// loads (lengths, list or table, stores): 4.9 us for 48 requests of one token, 6.2 us for 65,536 tokens of 64.
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

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef short s16x2 __attribute__((ext_vector_type(2)));

// Two packed bf16 over `scale` (a power of two) as e4m3 codes (nearest, ties to even; NaN as NaN; no more than 448 in
// magnitude), into the lower or the upper half of `into`. Equal to torch's conversion for every bf16 value.
template <bool UP>
__device__ __forceinline__ unsigned codes2(unsigned into, unsigned x, float scale) {
  return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(
                                          __builtin_bit_cast(s16x2, into), __builtin_bit_cast(bf16x2, x), scale, UP));
}
__device__ __forceinline__ unsigned codes4(unsigned x, unsigned y, float scale) {
  return codes2<true>(codes2<false>(0, x, scale), y, scale);
}
// Four codes under the scale `old` as codes under `scale`: rounded again (the elements are bf16 values).
__device__ __forceinline__ unsigned codes_again(unsigned w, float old, float scale) {
  return codes4(bf16_pair(w, old, false), bf16_pair(w, old, true), scale);
}

// The larger magnitudes, as bits, of packed bf16 pairs.
__device__ __forceinline__ unsigned larger(unsigned best, unsigned x) {
  return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(u16x2, best),
                                                                __builtin_bit_cast(u16x2, x & 0x7fff7fffu)));
}
// A pair with its infinities and NaN as zeros / with what is past `most` (a magnitude's bits) at `most`, NaN as it is.
__device__ __forceinline__ unsigned finite(unsigned x) {
  return ((x & 0x7fff) < 0x7f80 ? x & 0xffffu : 0u) | ((x >> 16 & 0x7fff) < 0x7f80 ? x & 0xffff0000u : 0u);
}
__device__ __forceinline__ unsigned at_most(unsigned x, unsigned most) {
  auto one = [&](unsigned v) {
    const unsigned m = v & 0x7fff;
    return m > most && m <= 0x7f80 ? (v & 0x8000) | most : v;
  };
  return one(x & 0xffff) | one(x >> 16) << 16;
}
// The maximum over the wave's lanes, in every lane.
__device__ __forceinline__ unsigned wave_largest(unsigned x) {
  // (as wave_scan: each lane's maximum with the lanes before it; lane 63 has all)
  auto step = [&](unsigned y) { x = max(x, y); };
  step(__builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));
  step(__builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));
  step(__builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));
  step(__builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));
  step(__builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));
  step(__builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));
  return __builtin_amdgcn_readlane(x, 63);
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
// merged (the block is this workgroup's alone). Bound by HBM: 32,768 rows of 16 heads at 128 86 us, 4.7 TB/s of rows read and
// codes written (97 us with the conversions one element at a time, 31 KB of code a kernel); by the launch and three rounds of
// dependent loads at a step's size: 6.7 us for one token of 48 requests.
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
  float* const scale_of = p.c.scales + 2 * head + (value ? 1 : 0);
  const unsigned old_bits = first > 0 ? __float_as_uint(*scale_of) : 0;

  // keys: tile i of the wave, token lane / 4 of its 16, elements (lane % 4) * 16 of its 64: x[2 i], x[2 i + 1]
  const int k_chunks = d >> 6;
  // values: lanes 8 i .. 8 i + 7 take tile i of the wave's 8; q = lane % 4, the tokens 16 t + 4 q + i as x[2 (4 t + i)] at
  // elements 8 * (lane / 4 % 2) .. + 8 and x[2 (4 t + i) + 1] 16 further on
  const int v_tile = wave * TILES + (lane >> 3), v_chunks = d >> 5;
  const int v_token = (v_tile / v_chunks) * 32 + (lane & 3) * 4, v_elem = (v_tile % v_chunks) * 32 + ((lane >> 2) & 1) * 8;
  const bool v_lane = (lane >> 3) < TILES;
  constexpr int kKeys = TILES * 2;
  u32x4 x[16];
  auto load = [&](int i, const uint16_t* src, bool mine) {
    x[i] = mine ? *reinterpret_cast<const u32x4*>(src) : u32x4{0, 0, 0, 0};
  };
  unsigned pair = 0;
  if (!value) {
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
      const int tile = wave * TILES + i, token = (tile / k_chunks) * 16 + (lane >> 2);
      const uint16_t* const src = in + token * stride + (tile % k_chunks) * 64 + (lane & 3) * 16;
      const bool mine = token >= first && token < first + count;
      load(2 * i, src, mine);
      load(2 * i + 1, src + 8, mine);
    }
#pragma unroll
    for (int i = kKeys; i < 16; ++i) x[i] = u32x4{0, 0, 0, 0};
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int token = v_token + (j >> 2) * 16 + (j & 3);
      const uint16_t* const src = in + token * stride + v_elem;
      const bool mine = v_lane && token >= first && token < first + count;
      load(2 * j, src, mine);
      load(2 * j + 1, src + 16, mine);
    }
  }
#pragma unroll
  for (int i = 0; i < 16; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) pair = larger(pair, x[i][j]);
  auto joined = [&](unsigned both) {  // over the workgroup
    unsigned best = wave_largest(max(both & 0xffffu, both >> 16));
    if constexpr (WAVES > 1) {
      __shared__ unsigned s_best[WAVES];
      __syncthreads();
      if (lane == 0) s_best[wave] = best;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < WAVES; ++w) best = max(best, s_best[w]);
    }
    return best;
  };
  unsigned best = joined(pair);
  const bool odd = best >= 0x7f80;  // infinities or NaN: the largest of the others
  if (__builtin_expect(odd, 0)) {
    pair = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) pair = larger(pair, finite(x[i][j]));
    best = joined(pair);
  }
  int e = exponent_of(best), old = e;
  if (first > 0) {
    old = min(max((int)((old_bits >> 23) & 0xff) - 127, KARPO_CACHE_MIN_EXP), KARPO_CACHE_MAX_EXP);
    e = max(e, old);
  }
  const bool grown = old < e;  // the earlier tokens' codes are rounded again
  const float scale = power_of_two(e), old_scale = power_of_two(old);
  if (threadIdx.x == 0) *scale_of = scale;
  if (__builtin_expect(odd || e == KARPO_CACHE_MAX_EXP, 0)) {
    const unsigned most = (unsigned)(e + 8 + 127) << 7 | 0x60;  // 448 * 2^e
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) x[i][j] = at_most(x[i][j], most);
  }

  if (!value) {
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
      const int tile = wave * TILES + i, token = (tile / k_chunks) * 16 + (lane >> 2);
      u32x4* const dst = reinterpret_cast<u32x4*>(out + tile * 1024 + lane * 16);
      if (token >= first && token < first + count) {
        const u32x4 a = x[2 * i], b = x[2 * i + 1];
        *dst = u32x4{codes4(a[0], a[1], scale), codes4(a[2], a[3], scale), codes4(b[0], b[1], scale),
                     codes4(b[2], b[3], scale)};
      } else if (grown && token < first) {
        u32x4 w = *dst;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = codes_again(w[j], old_scale, scale);
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
  u32x4 was[8];
  if (!whole) {
#pragma unroll
    for (int s = 0; s < 8; ++s) was[s] = dst[4 * s];
  }
#pragma unroll
  for (int s = 0; s < 8; ++s) {
    u32x4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // dh = j / 2, t = j % 2: element s of four tokens
      const int t = j & 1, dh = j >> 1;
      auto tokens = [&](int i) {
        return __builtin_amdgcn_perm(x[2 * (4 * t + i + 1) + dh][s >> 1], x[2 * (4 * t + i) + dh][s >> 1],
                                     s & 1 ? 0x07060302u : 0x05040100u);
      };
      w[j] = codes4(tokens(0), tokens(2), scale);
    }
    if (!whole) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned n = is_new[j & 1], o = is_old[j & 1];
        unsigned kept = was[s][j];
        if (grown) kept = (codes_again(kept, old_scale, scale) & o) | (kept & ~o);
        w[j] = (w[j] & n) | (kept & ~n);
      }
    }
    dst[4 * s] = w;
  }
}

// ---- read

constexpr int kReadWaves = 4;

// A wave takes 32 tokens of one head's keys or values at a time, the heads of a group one after the other, so that the rows
// that a workgroup writes lie side by side. Keys: 8 codes a lane make 16 bytes of a row, 8 lanes the 128 of a tile's row.
// Values: the tokens lie innermost, so the codes go through LDS (one tile after the other, 64 bytes between their halves
// against bank conflicts), out of which a lane takes 4 tokens x 8 elements: 16 bytes of four rows. Each workgroup adds up all
// lengths by itself and takes an equal share of all groups. Bound by HBM: 32,768 rows of 16 heads at 128 72 us, 5.6 TB/s; 9,244
// rows of 4 heads at 512 19.8 us, 5.7 TB/s (112 and 36.6 us with 8-byte stores of the values and a head a workgroup).
template <int D, bool STREAM>
__global__ __launch_bounds__(64 * kReadWaves) void read_kernel(const ReadParams p) {
  constexpr int kThreads = 64 * kReadWaves, kTiles = D / 32;
  constexpr int kAtOnce = kTiles < 4 ? kTiles : 4;  // KiB of codes that a lane's loads have in flight
  constexpr int kTileBytes = 2 * (512 + 64);
  __shared__ int s_part[kReadWaves][2];
  __shared__ int s_group[kThreads + 1], s_row[kThreads], s_start[kThreads], s_tokens[kThreads];
  __shared__ __align__(16) char s_codes[kReadWaves][kAtOnce * kTileBytes];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int heads = p.c.kv_heads, b = p.c.block_log2;

  // first and last token of request i that are read
  bool bad = false;  // (with q_cu) bounds that the attention's planner refuses
  auto range = [&](int i, int* start, int* tokens) {
    *tokens = min(max(p.r.lengths[i], 0), p.r.most);
    *start = 0;
    if (p.q_cu != nullptr) {
      const int q0 = p.q_cu[i], q1 = p.q_cu[i + 1];
      const int64_t queries = (int64_t)q1 - q0;
      bad |= q0 < 0 || queries < 0 || queries > p.max_q || q1 > p.total_q;
      if (queries <= 0) {
        *tokens = 0;
      } else if (p.window_left >= 0) {
        const int64_t s = (int64_t)*tokens - queries - p.window_left;
        *start = s > 0 ? (int)ka_min64(s, *tokens) & ~(kCacheGroup - 1) : 0;
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
  int groups = 0;
  int64_t rows = 0;
  for (int c0 = 0; c0 < p.r.n_seq; c0 += kThreads) {
    if (c0 > 0) __syncthreads();
    scan(c0);
    groups += all[0];
    rows += (int64_t)all[0] * kCacheGroup + all[1];
  }
  if (p.q_cu != nullptr && __syncthreads_or(bad || rows > p.rows || p.no_scale)) {
    for (int i = 0; i < p.r.n_seq; ++i) {
      const int q0 = p.q_cu[i], q1 = p.q_cu[i + 1];
      if (q0 >= 0 && q1 > q0 && q1 <= p.total_q)
        fill_rows<D>(p.no_scale && p.r.lengths[i] <= 0 ? 0u : kNanPair, p.o + q0 * p.so_t, p.so_t, p.so_h, q1 - q0, p.heads,
                     (int64_t)blockIdx.x * kThreads + tid, (int64_t)gridDim.x * kThreads);
    }
  }
  auto store = [&](uint16_t* to, const u32x4& x) {
    if constexpr (STREAM) __builtin_nontemporal_store(x, reinterpret_cast<u32x4*>(to)); else *reinterpret_cast<u32x4*>(to) = x;
  };
  // units: (group, head, keys or values, kAtOnce tiles of them)
  constexpr int kPieces = kTiles / kAtOnce;
  const int sides = 2 * heads * kPieces;
  const int64_t units = (int64_t)groups * sides;
  const int64_t u0 = units * blockIdx.x / gridDim.x, u1 = units * (blockIdx.x + 1) / gridDim.x;

  int carry_groups = 0;
  int64_t carry_rows = 0;
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
    if (blockIdx.x == 0 && i < p.r.n_seq) p.k_cu[i] = (int)ka_min64(row, INT32_MAX);
    __syncthreads();
    const int64_t chunk0 = (int64_t)carry_groups * sides, from = u0 > chunk0 ? u0 : chunk0;
    const int64_t to = ka_min64(u1, chunk0 + (int64_t)all[0] * sides);
    int token0 = 0, tokens_left = 0, id = 0, group = -1;
    int64_t out_row = 0;
    int g = (int)(from / sides), side = (int)(from - (int64_t)g * sides) + wave;
    for (int64_t unit = from + wave; unit < to; unit += kReadWaves, side += kReadWaves) {
      for (; side >= sides; side -= sides) ++g;
      const int h = side / (2 * kPieces), t0 = (side % kPieces) * kAtOnce;
      const bool value = (side / kPieces) & 1;
      if (g != group) {
        group = g;
        const int u = g - carry_groups;
        const int j = last_at_most(s_group, m, u);
        token0 = s_start[j] + (u - s_group[j]) * kCacheGroup;
        out_row = (int64_t)s_row[j] + token0 - s_start[j];
        tokens_left = (int)ka_min64(ka_min64(s_tokens[j] - token0, p.rows - out_row), kCacheGroup);
        id = p.r.table[(int64_t)(c0 + j) * p.r.table_stride + (token0 >> b)];
      }
      if (tokens_left <= 0) continue;
      const bool known = id >= 0 && id < p.c.blocks;
      const int64_t head = (int64_t)(known ? id : 0) * heads + h;
      const int inside = token0 & ((1 << b) - 1);
      const uint8_t* const src = (value ? p.c.values : p.c.keys) + (head << b) * D + inside * D;
      const float scale = known ? p.c.scales[2 * head + (value ? 1 : 0)] : 1.f;  // (zeros under any other block's could be NaN)
      uint16_t* const dst = (value ? p.v : p.k) + (out_row * heads + h) * D;
      const int64_t step = (int64_t)heads * D;
      if (!value) {
        constexpr int kChunks = D / 64;  // tiles of 16 tokens x 64 elements, each in two halves of 8 tokens
        u32x2 w[2 * kAtOnce];
#pragma unroll
        for (int t = 0; t < 2 * kAtOnce; ++t)
          w[t] = known ? *reinterpret_cast<const u32x2*>(src + (2 * t0 + t) * 512 + lane * 8) : u32x2{0, 0};
#pragma unroll
        for (int t = 0; t < 2 * kAtOnce; ++t) {
          const int tile = t0 + (t >> 1), token = (tile / kChunks) * 16 + (t & 1) * 8 + (lane >> 3);
          if (token < tokens_left)
            store(dst + token * step + (tile % kChunks) * 64 + (lane & 7) * 8, bf16_of_8(w[t][0], w[t][1], scale));
        }
      } else {
        // of each two tiles: lane = (dlow half, dh, tile of the two, t, q): elements 16 dh + 8 (dlow half) + 0 .. 7 of the tile
        const int half = lane & 1, dh = (lane >> 1) & 1, which = (lane >> 2) & 1, t16 = (lane >> 3) & 1, q = lane >> 4;
        char* const codes = s_codes[wave];
        u32x4 w[kAtOnce];
#pragma unroll
        for (int t = 0; t < kAtOnce; ++t)
          w[t] = known ? *reinterpret_cast<const u32x4*>(src + (t0 + t) * 1024 + lane * 16) : u32x4{0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < kAtOnce; ++t)
          *reinterpret_cast<u32x4*>(codes + t * kTileBytes + (lane >> 5) * (512 + 64) + (lane & 31) * 16) = w[t];
#pragma unroll
        for (int t = 0; t < kAtOnce; t += 2) {
          const char* const from_codes =
              codes + (t + which) * kTileBytes + half * (512 + 64) + q * 16 + dh * 8 + t16 * 4;
          unsigned pair[2][8];  // tokens 0, 1 and 2, 3 of the four, of each element
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const unsigned c = *reinterpret_cast<const unsigned*>(from_codes + e * 64);
            pair[0][e] = bf16_pair(c, scale, false);
            pair[1][e] = bf16_pair(c, scale, true);
          }
          const int token = 16 * t16 + 4 * q;
          uint16_t* const to_row = dst + token * step + (t0 + t + which) * 32 + dh * 16 + half * 8;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const unsigned(&x)[8] = pair[e >> 1];
            const unsigned pick = e & 1 ? 0x07060302u : 0x05040100u;
            if (token + e < tokens_left)
              store(to_row + e * step,
                    u32x4{__builtin_amdgcn_perm(x[1], x[0], pick), __builtin_amdgcn_perm(x[3], x[2], pick),
                        __builtin_amdgcn_perm(x[5], x[4], pick), __builtin_amdgcn_perm(x[7], x[6], pick)});
          }
        }
      }
    }
    carry_groups += all[0];
    carry_rows += (int64_t)all[0] * kCacheGroup + all[1];
    __syncthreads();
  }
  if (blockIdx.x == 0 && tid == 0) p.k_cu[p.r.n_seq] = (int)ka_min64(carry_rows, INT32_MAX);
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
  // A unit each wave, at most 32 workgroups per CU: 32,768 rows of 16 heads at 128 96.9 us with 1,024 workgroups, 85.5 with
  // 2,048, 82.0 with 4,096, 77.6 with 8,192 (how evenly the rows being written lie over the memory's channels; measured before
  // such rows were stored through the caches, 72 us since).
  const int64_t units = (p.rows / kCacheGroup + p.r.n_seq) * 2 * p.c.kv_heads * (p.c.head_dim == 64 ? 1 : p.c.head_dim / 128);
  const dim3 grid((unsigned)ka_min64((units + kReadWaves - 1) / kReadWaves + 1, 8192)), threads(64 * kReadWaves);
  auto launch = [&](auto d) {
    constexpr int D = decltype(d)::value;
    if (p.stream) read_kernel<D, true><<<grid, threads, 0, stream>>>(p); else read_kernel<D, false><<<grid, threads, 0, stream>>>(p);
  };
  switch (p.c.head_dim) {
    case 64: launch(std::integral_constant<int, 64>()); break;
    case 128: launch(std::integral_constant<int, 128>()); break;
    case 256: launch(std::integral_constant<int, 256>()); break;
    case 512: launch(std::integral_constant<int, 512>()); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace karpo
