// Attention over the block cache in 4 bits for few queries per request (karpo_cache4_attend): the keys of all requests are split
// over the workgroups that the GPU holds at once, 32 tokens at a time, and the shares of a request joined by a second launch.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "cache.h"
#include "cache_attn_common.h"

namespace karpo {

namespace {

// Waves per SIMD (and workgroups per CU): what the registers hold without spilling; attend4_kernel<128, 4> alone spills 7, four of
// which each group loads again.
__host__ __device__ constexpr int attend4_waves(int d, int nt) {
  return nt == 1 ? (d == 64 ? 4 : d == 128 ? 3 : d == 256 ? 2 : 1) : d == 64 && nt == 2 ? 3 : d <= 128 ? 2 : 1;
}
// Bytes of LDS for the waves' copies of a group's keys (as many for the values).
constexpr int ring4_bytes(int d, int waves) { return waves * kCacheGroup * d / 2; }
// And for their sums while they are joined.
constexpr int sums4_bytes(int d, int nt, int waves) { return waves * 16 * nt * (slab_of(d, nt) + 4) * 4; }

// Requests of which at most so many tokens are seen (by the bounds that the call gives, the table's width among them) are not
// split: a workgroup's walk is then shorter than the partials' way through memory and a second launch. us split, whole by four
// waves at heads of 128 with 16 key heads: 8 requests of 128 tokens 12.4, 7.3, of 640 15.9, 11.4, of 1,500 18.9, 18.7; one of
// 1,024 13.7, 13.6; heads of 512, 2 requests of 256 15.8, 13.0, of 512 16.7, 17.6. The bound is that of four waves. Where eight
// would walk (AttendShape::wide) they are faster past it too: 8 requests of 1,000 tokens, 16 heads of 128 17.4, 12.6, 2 of 64
// 13.4, 10.3, 8 of 256 18.0, 16.0; of 1,300 18.4, 14.1; 13.7, 11.6; 19.3, 18.1; one of 1,300, 16 heads of 128 13.9, 12.9, 8 of
// 256 15.7, 17.2.
constexpr int whole_tokens4(int d) { return d == 512 ? 256 : 640; }
// Where more than half of the CUs have a workgroup, a longer walk is no loss (48 requests of 4 query tokens and 1,024 cached
// ones: heads of 64 18.4, 13.0; 128 33.4, 27.4; 256 36.1, 29.9; 512 64.4, 60.5), up to what one long request among short ones
// may take: one of 1,280 seen tokens 12.5 to 20 us, of heads of 512 30, against 13.5 to 19 and 23 where its shares are split.
constexpr int most_whole_tokens4(int d) { return d == 512 ? 1024 : 1280; }
constexpr int kLeastUnits4 = 4;         // groups of 32 tokens that a workgroup takes at least, of a request that is split

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef short s16x2 __attribute__((ext_vector_type(2)));

// acc + (16 keys x 128 elements of e2m1 codes, with byte KB of the lane's word of scales) x (e4m3 terms of 16 query vectors,
// with byte QB of theirs).
template <int KB, int QB>
__device__ __forceinline__ f32x4 mfma_codes4(const u32x4& k, unsigned k_scale, const u32x4& q0, const u32x4& q1, unsigned q_scale,
                                             f32x4 acc) {
  const i32x8 a = {(int)k[0], (int)k[1], (int)k[2], (int)k[3], 0, 0, 0, 0};
  const i32x8 b = {(int)q0[0], (int)q0[1], (int)q0[2], (int)q0[3], (int)q1[0], (int)q1[1], (int)q1[2], (int)q1[3]};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 0, KB, (int)k_scale, QB, (int)q_scale);
}

constexpr int kMostQueryExp = 120;  // of the scale of 32 of a query's elements: that of those past 448 * 2^119

// 16 bf16 over 2^e as 16 e4m3 codes, and what they leave over (exact in fp32) over 2^(e - 4). Finite elements from 248 * 2^120 on
// would round to 256 * 2^120, which neither bf16 nor a sum of fp32 holds: their first term is 240 * 2^120, and the second the rest
// (8 to 15, 128 to 240 of its own scale's, which have steps of 16: exact).
__device__ __forceinline__ void two_terms(const u32x4 (&x)[2], int e, u32x4* high, u32x4* low) {
  const float scale = power_of_two(e), fine = power_of_two(e - 4);
  const bool largest = __any(e == kMostQueryExp);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    float v[4], h[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = bf16_at(x[w >> 1], (w & 1) * 4 + k);
#pragma unroll
    for (int k = 0; k < 4; ++k) h[k] = v[k];
    if (__builtin_expect(largest, 0)) {
      constexpr float kMost = 240.f * 0x1p120f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float m = __builtin_fabsf(v[k]);
        h[k] = m > kMost && m < INFINITY ? __builtin_copysignf(kMost, v[k]) : v[k];
      }
    }
    s16x2 c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(s16x2{0, 0}, h[0], h[1], scale, false);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, h[2], h[3], scale, true);
    (*high)[w] = __builtin_bit_cast(unsigned, c);
#pragma unroll
    for (int k = 0; k < 4; k += 2) {
      const unsigned back = bf16_pair((*high)[w], scale, k != 0);
      h[k] = __uint_as_float(back << 16);
      h[k + 1] = __uint_as_float(back & 0xffff0000u);
    }
    c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(s16x2{0, 0}, v[0] - h[0], v[1] - h[1], fine, false);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, v[2] - h[2], v[3] - h[3], fine, true);
    (*low)[w] = __builtin_bit_cast(unsigned, c);
  }
}

// Two e2m1 codes, byte BYTE of `w`, under the scale with these exponent bits, as packed bf16.
template <int BYTE>
__device__ __forceinline__ unsigned pair_at(unsigned w, unsigned scale) {
  return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, __uint_as_float(scale), BYTE));
}

// How the requests' groups lie on a line that the workgroups cut into equal pieces: request i takes `weight(units)` of it, its
// groups first. Where the pieces of whole requests, ceil(units / each) of them, are no more than the workgroups, a request begins
// at a piece's begin (`start` < 0) and no workgroup changes its request; otherwise a workgroup may go on to a next request, and
// spends about as long on the change (joining its waves, the new queries and table, the first copies) as on `start` groups.
struct Line {
  int each, more, start;
  __device__ __forceinline__ int weight(int units) const {
    return start < 0 ? (int)((unsigned)(units + each - 1) / (unsigned)each) * each : units > 0 ? units + start : 0;
  }
  __device__ __forceinline__ int begin(int part) const { return part * each + min(part, more); }
  __device__ __forceinline__ int part_of(int unit) const {
    const int longer = more * (each + 1);
    return unit < longer ? (int)((unsigned)unit / (unsigned)(each + 1)) : more + (int)((unsigned)(unit - longer) / (unsigned)each);
  }
};
// 48 requests, 16 heads of 128: kStart4 of 8, 12, 16, 24 groups 40.0, 37.6, 37.1, 38.2 us. kTries: lengths of pieces that are tried.
constexpr int kStart4 = 16, kTries = 5;

// As in the kernel over 8 bits: S^T = K Q^T with keys as rows, a lane's eight weights (keys 16 t + 4 (lane / 16) + i of column
// lane % 16) as they stand the second operand of O^T = V^T P^T; a wave takes every fourth group of 32 tokens by itself, the
// next group's keys on their way to LDS while this one's weights are made, the next values while the next keys are read; the
// weights enter the second product as two bf16 terms.
//
// The keys' codes are the first operand of S^T as they come out of the cache (16x16x128 scaled matrix instructions: 16 tokens
// x 128 elements, a lane's 32 elements under their own scale), the queries the second, as two e4m3 terms (8 significant bits, a
// bf16's, for elements within 2^-14 of the largest of their 32; 2^-22 of that largest otherwise). A value's scale is its token's,
// and tokens are what the second product sums over, so values become bf16 in registers: two elements of a token a conversion,
// two tokens' of an element a permutation. Of head size 64 a lane's operand holds two tiles of 16 tokens, and the queries fill
// its one half or the other.
//
// Bound by HBM: one request of 131,073 tokens, 32 / 4 heads of 512, 55 us for 285 MB (5.2 TB/s; the walk itself at 6 to 7, its start
// and end take 5 to 7 us together), 48 requests of 68,664 together, 32 / 16 of 128, 37 us for 150 MB, of which the start, the changes
// from request to request (2 us each) and the unequal ends are 14. The matrix units are busy for 19 and 15% of that. Deeper rings,
// groups of 64 tokens and four waves a SIMD at head size 128 (42.3 against 40.1 us) were no faster.
//
// ONCE: one workgroup reads a request's codes of a head, once; they are streamed through the caches.
template <int D, int NT, bool ONCE, int WAVES>
__device__ __forceinline__ void attend4_share(const AttendParams& p, const Seen& s, int request, int g0, int g1, int h,
                                              int vector0, int vectors, bool whole, float* part) {
  constexpr int kGroupBytes = kCacheGroup * D / 2;
  constexpr int kLoads = kGroupBytes / 1024;  // KiB of keys, and of values, in a group
  constexpr int kCopies = kLoads + 1;         // with their scales
  constexpr int kSpans = D < 128 ? 1 : D / 128, kParts = D < 128 ? 1 : 2;  // spans of 128 elements, two pieces of 64 each
  constexpr int kGroups = D / 32;                                          // of 32 elements under a scale
  constexpr int kSlab = slab_of(D, NT), kVectors = 16 * NT;
  constexpr int kRing = ring4_bytes(D, WAVES);
  __shared__ float s_m[WAVES][kVectors], s_l[WAVES][kVectors];
  // (arrays of their own: a read then waits for the copies into its own array and no others)
  __shared__ __align__(16) char s_keys[kRing > sums4_bytes(D, NT, WAVES) ? kRing : sums4_bytes(D, NT, WAVES)];
  __shared__ __align__(16) char s_values[kRing];
  __shared__ __align__(16) char s_key_scales[WAVES * 1024], s_value_scales[WAVES * 1024];  // (D bytes each in use)
  __shared__ u32x4 s_q[kVectors * D / 8];
  __shared__ unsigned s_q_scales[kSpans * NT * 64];
  float(*const s_o)[kVectors][kSlab + 4] = reinterpret_cast<float(*)[kVectors][kSlab + 4]>(s_keys);
  // (a request's addresses are made anew for each: kept over the walk of requests, they and what spills for them cost 15 to 70
  // registers)
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, quad = lane >> 4;
  KA_LDS char* const key_ring = (KA_LDS char*)s_keys + wave * kGroupBytes;
  KA_LDS char* const value_ring = (KA_LDS char*)s_values + wave * kGroupBytes;
  KA_LDS char* const key_scales = (KA_LDS char*)s_key_scales + wave * 1024;
  KA_LDS char* const value_scales = (KA_LDS char*)s_value_scales + wave * 1024;
  const int heads = p.c.kv_heads, b = p.c.block_log2;

  // the query vectors' elements (a wave's spans of them: 16 quad .. + 16 of each 64), and the keys that each vector sees
  constexpr int kMine = (kSpans * NT + WAVES - 1) / WAVES;
  u32x4 q_mine[kMine][2 * kParts];
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
      const int e = wave + c * WAVES;  // span e / NT of tile e % NT
      if (e < kSpans * NT && e % NT == n) {
#pragma unroll
        for (int k = 0; k < 2 * kParts; ++k)
          q_mine[c][k] = *reinterpret_cast<const u32x4*>(src + (e / NT) * 128 + (k >> 1) * 64 + quad * 16 + (k & 1) * 8);
      }
    }
    lo[n] = p.left < 0 ? 0 : pos + shift - p.left;
    hi[n] = p.right < 0 ? s.tokens - 1 : (int)min<int64_t>((int64_t)pos + shift + p.right, s.tokens - 1);
  }
  // groups that every vector sees whole
  const int pos_first = position_of(vector0, p), pos_last = position_of(vector0 + vectors - 1, p);
  const int full_lo = p.left < 0 ? 0 : pos_last + shift - p.left;
  const int full_hi = p.right < 0 ? s.tokens - 1 : (int)min<int64_t>((int64_t)pos_first + shift + p.right, s.tokens - 1);
  // tokens that any vector sees
  const int any_lo = p.left < 0 ? 0 : pos_first + shift - p.left;
  const int any_hi = p.right < 0 ? s.tokens - 1 : (int)min<int64_t>((int64_t)pos_last + shift + p.right, s.tokens - 1);

  f32x4 o[NT][D / 16];  // [2 (32 elements) + which of each pair of them]
  float top[NT], sum[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    top[n] = -INFINITY;
    sum[n] = 0.f;
#pragma unroll
    for (int t = 0; t < D / 16; ++t) o[n][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const int32_t* const table = p.r.table + (int64_t)request * p.r.table_stride;
  int ids = 0;
  // lane k looks up the wave's groups g + 4 k
  auto look_up = [&](int g) {
    ids = table[min(g + lane * WAVES, g1 - 1) >> (b - 5)];
    if (ids < 0 || ids >= p.c.blocks) ids = -1;
  };
  // One group's codes and scales into the wave's ring, 16 bytes a lane; zeros for a block that is not of the pool (and for the
  // lanes past the scales, which all take part so that a wait can count the copies).
  auto copy = [&](bool value, int g, int k) {
    const int id = __builtin_amdgcn_readlane(ids, k & 63);
    const int64_t head = (int64_t)max(id, 0) * heads + h;
    const int64_t token = (head << b) + (int64_t)(g & ((1 << (b - 5)) - 1)) * kCacheGroup;
    const __amdgpu_buffer_rsrc_t r =
        __builtin_amdgcn_make_buffer_rsrc((void*)((value ? p.c.values : p.c.keys) + token * (D / 2)), (short)0,
                                          id >= 0 ? kGroupBytes : 0, kBufferFlags);
    KA_LDS char* const to = value ? value_ring : key_ring;
#pragma unroll
    for (int t = 0; t < kLoads; ++t)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (KA_LDS void*)(to + t * 1024), 16, lane * 16, t * 1024, 0,
                                               ONCE ? kCopyStream : 0);
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
        (void*)(p.c.scales4 + token * (D / 16) + (value ? D : 0)), (short)0, id >= 0 ? D : 0, kBufferFlags);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (KA_LDS void*)(value ? value_scales : key_scales), 16, lane * 16, 0, 0, 0);
  };
  auto tile = [&](const KA_LDS char* ring, int t) {
    return *reinterpret_cast<const KA_LDS u32x4*>(ring + t * 1024 + lane * 16);
  };
  // this lane's tokens' scales of 32 elements of the values: bytes 4 t + i
  auto scales_at = [&](int group) { return reinterpret_cast<KA_LDS u32x2*>(value_scales + group * 32 + quad * 8); };
  // all but the last issued group's keys, or values, have arrived / the reads of the ring are done
  auto arrived = [&]() {
    wait_vmcnt<kCopies>();
    asm volatile("" ::: "memory");
  };
  auto read_out = [&]() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); };

  int k = 0;
  const bool some = g0 + wave < g1;
  if (some) {  // on their way while the queries are made
    look_up(g0 + wave);
    copy(false, g0 + wave, 0);
    copy(true, g0 + wave, 0);
  }
#pragma unroll
  for (int c = 0; c < kMine; ++c) {
    const int e = wave + c * WAVES;
    if (e < kSpans * NT) {
      // the largest of each 32 elements: of a lane's 16 and those of the lane 16 away; 448 * 2^e holds it
      int part_e[2] = {0, 0};
#pragma unroll
      for (int j = 0; j < kParts; ++j) {
        unsigned m = 0;
#pragma unroll
        for (int w = 0; w < 8; ++w) {
          const unsigned x = q_mine[c][2 * j + (w >> 2)][w & 3];
          m = max(m, max(x & 0x7fff, x >> 16 & 0x7fff));
        }
        m = max(m, (unsigned)__shfl_xor((int)m, 16));
        part_e[j] = min(max((int)(m >> 7) - 127 - 8 + ((m & 0x7f) > 0x60 ? 1 : 0), -100), kMostQueryExp);
      }
      // the scales go by 32 elements in order, which these lanes have
      const int from = col + 16 * ((2 * quad) & 3);
      const int first = __shfl(part_e[0], from), second = kParts == 2 ? __shfl(part_e[1], from) : first;
      const int mine_e = kParts == 1 || quad < 2 ? first : second;
      s_q_scales[e * 64 + lane] = (unsigned)(mine_e + 127) | (unsigned)(mine_e - 4 + 127) << 8;
#pragma unroll
      for (int j = 0; j < kParts; ++j) {
        const u32x4 x[2] = {q_mine[c][2 * j] ^ p.sign, q_mine[c][2 * j + 1] ^ p.sign};
        u32x4 high, low;
        two_terms(x, part_e[j], &high, &low);
        s_q[((e * 2 + 0) * kParts + j) * 64 + lane] = high;
        s_q[((e * 2 + 1) * kParts + j) * 64 + lane] = low;
      }
    }
  }
  lds_barrier();
  for (int g = g0 + wave; g < g1; g += WAVES) {
    const int next = g + WAVES;
    arrived();
    f32x4 st[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) st[n][0] = st[n][1] = f32x4{0.f, 0.f, 0.f, 0.f};
    {
      constexpr int kWords = D < 256 ? 1 : D / 256;  // of a lane's scales of its group
      unsigned ks[kWords];
      const KA_LDS char* const from = key_scales + lane * (D / 64);
      if constexpr (D == 64) ks[0] = *reinterpret_cast<const KA_LDS uint8_t*>(from);
      if constexpr (D == 128) ks[0] = *reinterpret_cast<const KA_LDS uint16_t*>(from);
      if constexpr (D == 256) ks[0] = *reinterpret_cast<const KA_LDS unsigned*>(from);
      if constexpr (D == 512) {
        const u32x2 w = *reinterpret_cast<const KA_LDS u32x2*>(from);
        ks[0] = w[0];
        ks[kWords - 1] = w[1];
      }
      const u32x4 none = {0, 0, 0, 0};
#pragma unroll
      for (int dt = 0; dt < kSpans; ++dt)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int entry = dt * NT + n;
          const unsigned qs = s_q_scales[entry * 64 + lane];
          u32x4 q[2][2];  // [term][piece]
#pragma unroll
          for (int term = 0; term < 2; ++term)
#pragma unroll
            for (int j = 0; j < kParts; ++j) q[term][j] = s_q[((entry * 2 + term) * kParts + j) * 64 + lane];
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const u32x4 a = tile(key_ring, D == 64 ? 0 : t * kSpans + dt);
            f32x4& acc = st[n][t];
            // (of head size 64 the other tile's tokens meet zeros, which a NaN scale of theirs would make NaN)
            const unsigned k_scale = D == 64 && quad >> 1 != t ? 0u : ks[dt >> 1];
            const u32x4 h0 = D == 64 && t == 1 ? none : q[0][0], h1 = D == 64 ? (t == 1 ? q[0][0] : none) : q[0][1];
            const u32x4 l0 = D == 64 && t == 1 ? none : q[1][0], l1 = D == 64 ? (t == 1 ? q[1][0] : none) : q[1][1];
            auto add = [&](auto byte) {
              constexpr int KB = decltype(byte)::value;
              acc = mfma_codes4<KB, 0>(a, k_scale, h0, h1, qs, acc);
              acc = mfma_codes4<KB, 1>(a, k_scale, l0, l1, qs, acc);
            };
            if (D == 64 || (2 * dt + t) % 4 == 0) add(std::integral_constant<int, 0>());
            else if ((2 * dt + t) % 4 == 1) add(std::integral_constant<int, 1>());
            else if ((2 * dt + t) % 4 == 2) add(std::integral_constant<int, 2>());
            else add(std::integral_constant<int, 3>());
          }
        }
    }
    read_out();
    if (++k == 64 && next < g1) {
      look_up(next);
      k = 0;
    }
    if (next < g1) copy(false, next, k);

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
      // what the weights are taken against is raised (and O rescaled) only where a score passes it, and then to 2^8 above the
      // largest: weights are at most 1, and sums of the largest values within fp32's range, as in the formula
      if (__any(!(best <= top[n]) && best != -INFINITY)) {
        const float up = __builtin_elementwise_maximum(top[n], best + 8.f);
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
        low[e] = pair_of(w[2 * e] - __uint_as_float(high[e] << 16), w[2 * e + 1] - __uint_as_float(high[e] & 0xffff0000u));
      }
      weight[n][0] = __builtin_bit_cast(bf16x8, high);
      weight[n][1] = __builtin_bit_cast(bf16x8, low);
      sum[n] += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
    }

    if (next < g1) arrived(); else wait_vmcnt<0>();
    asm volatile("" ::: "memory");
    bool odd = false;
    if (masked) {
      unsigned any = 0;  // 0x80 where a byte is 253 (KARPO_CACHE4_MAX_EXP + 128) or more
#pragma unroll
      for (int group = 0; group < kGroups; ++group) {
        const u32x2 w = *scales_at(group);
#pragma unroll
        for (int t = 0; t < 2; ++t) any |= ((w[t] & 0x7f7f7f7fu) + 0x03030303u) & w[t] & 0x80808080u;
      }
      odd = __any(any != 0);
    }
    // a NaN reaches the vectors that see its token, and no others, and what a slot holds that nothing wrote (253 and 254: codes
    // under them pass bf16's range) reaches none (zero times NaN or infinity would be NaN)
    if (odd) {
      unsigned hidden = 0;  // one bit of each of the lane's eight keys that no vector sees
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int key = key0 + (e >> 2) * 16 + quad * 4 + (e & 3);
        hidden |= key < any_lo || key > any_hi ? 1u << e : 0u;
      }
#pragma unroll
      for (int group = 0; group < kGroups; ++group) {
        u32x2 w = *scales_at(group);
        unsigned marks = 0;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool nan = (w[t] >> (8 * i) & 255) == 255;
            marks |= nan ? 1u << (4 * t + i) : 0u;
            if (nan || (hidden >> (4 * t + i) & 1) != 0) w[t] &= ~(255u << (8 * i));
          }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float hit = column_sum((is_seen[n] & marks) != 0 ? 1.f : 0.f);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            o[n][2 * group][e] += hit > 0.f ? NAN : 0.f;
            o[n][2 * group + 1][e] += hit > 0.f ? NAN : 0.f;
          }
        }
        *scales_at(group) = w;  // (every lane of the quad the same: what a lane read before, it may not keep)
      }
    }
#pragma unroll
    for (int t64 = 0; t64 < kLoads; ++t64) {
      const u32x4 w = tile(value_ring, t64);
#pragma unroll
      for (int d = 0; d < 2; ++d) {
        const int group = 2 * t64 + d;
        const u32x2 sc = *scales_at(group);
        u32x4 even, odd;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          // (the conversion goes by its scale's exponent bits alone, 30 .. 23)
          const unsigned c = w[2 * d + t];
          const unsigned r0 = pair_at<0>(c, sc[t] << 23), r1 = pair_at<1>(c, sc[t] << 15);
          const unsigned r2 = pair_at<2>(c, sc[t] << 7), r3 = pair_at<3>(c, sc[t] >> 1);
          even[2 * t] = __builtin_amdgcn_perm(r1, r0, 0x05040100u);
          even[2 * t + 1] = __builtin_amdgcn_perm(r3, r2, 0x05040100u);
          odd[2 * t] = __builtin_amdgcn_perm(r1, r0, 0x07060302u);
          odd[2 * t + 1] = __builtin_amdgcn_perm(r3, r2, 0x07060302u);
        }
        const bf16x8 a = __builtin_bit_cast(bf16x8, even), c = __builtin_bit_cast(bf16x8, odd);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int term = 0; term < 2; ++term) {
            o[n][2 * group] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, weight[n][term], o[n][2 * group], 0, 0, 0);
            o[n][2 * group + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(c, weight[n][term], o[n][2 * group + 1], 0, 0, 0);
          }
      }
    }
    read_out();
    if (next < g1) copy(true, next, k);
  }

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
    for (int w = 1; w < WAVES; ++w) up = __builtin_elementwise_maximum(up, s_m[w][c]);
    return up;
  };
  auto total_of = [&](int c, float up) {
    float l = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w)
      l += s_m[w][c] == -INFINITY ? 0.f : s_l[w][c] * __builtin_amdgcn_exp2f(s_m[w][c] - up);
    return l;
  };
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
      for (int t = 0; t < D / 16; t += 2)
        if (t * 16 >= d0 && t * 16 < d0 + kSlab) {
          const f32x4 a = o[n][t] * f, c = o[n][t + 1] * f;
          f32x4* const to = reinterpret_cast<f32x4*>(&s_o[wave][16 * n + col][t * 16 - d0 + quad * 8]);
          to[0] = f32x4{a[0], c[0], a[1], c[1]};
          to[1] = f32x4{a[2], c[2], a[3], c[3]};
        }
    }
    lds_barrier();
    for (int e = tid; e < vectors * (kSlab / 4); e += 64 * WAVES) {
      const int c = e / (kSlab / 4), d = (e % (kSlab / 4)) * 4;
      f32x4 x = *reinterpret_cast<const f32x4*>(&s_o[0][c][d]);
#pragma unroll
      for (int w = 1; w < WAVES; ++w) x += *reinterpret_cast<const f32x4*>(&s_o[w][c][d]);
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

template <int D, int NT, bool ONCE>
__global__ __launch_bounds__(kAttendThreads, attend4_waves(D, NT)) void attend4_kernel(const AttendParams p) {
  constexpr int kVectors = 16 * NT;
  __shared__ int s_part[kAttendWaves][2], s_try[kAttendWaves][kTries], s_sum[kAttendWaves][1];
  __shared__ Seen s_seen;
  __shared__ int s_at[2];
  const int tid = threadIdx.x;
  const int heads = p.c.kv_heads;
  const int h = blockIdx.y % heads, vector0 = (blockIdx.y / heads) * kVectors;

  // a chunk of requests, one a thread, and this workgroup's piece u0 .. u1 of the line
  Seen own;
  int v[1] = {0}, all[1];
  Line line = {1, 0, -1};
  auto take = [&](int c0) {
    own = Seen{0, 0, 0, 0, 0, 0};
    if (c0 + tid < p.r.n_seq) own = seen_of(p, c0 + tid);
  };
  int c0 = 0, u0, u1;
  int units = 0, requests = 0;
  for (int c = 0; c < p.r.n_seq; c += kAttendThreads) {
    if (c > 0) __syncthreads();
    take(c);
    int w[2] = {own.units, own.units > 0 ? 1 : 0}, sums[2];
    block_scan<kAttendThreads, 2>(w, sums, s_part);
    units += sums[0];
    requests += sums[1];
  }
  const int least = max(kLeastUnits4, (int)((unsigned)(units + p.parts - 1) / (unsigned)p.parts));
  const int total = max(units + (requests - 1) * kStart4, 0);  // (none comes after the last)
  const int most = max(least, (int)((unsigned)total / (unsigned)p.parts) + 1);
  if (p.r.n_seq <= kAttendThreads) {
    // the shortest pieces, from `least` to `most`, of which whole requests have no more than there are workgroups
    int w[kTries], sums[kTries];
#pragma unroll
    for (int t = 0; t < kTries; ++t) {
      const int each = least + (most - least) * t / (kTries - 1);
      w[t] = (int)((unsigned)(own.units + each - 1) / (unsigned)each);
    }
    block_scan<kAttendThreads, kTries>(w, sums, s_try);
    line.each = 0;
#pragma unroll
    for (int t = kTries - 1; t >= 0; --t)
      if (sums[t] <= p.parts) line.each = least + (most - least) * t / (kTries - 1);
  } else {
    line.each = 0;
  }
  int end;  // of the line
  if (line.each > 0) {
    end = p.parts * line.each;
  } else {
    const unsigned n = max(min(p.parts, total / kLeastUnits4), 1);
    line = Line{(int)((unsigned)total / n), 0, kStart4};
    line.more = total - line.each * (int)n;
    end = total;
  }
  u0 = min(line.begin(blockIdx.x), end);  // (workgroups past the pieces: none)
  u1 = min(line.begin(blockIdx.x + 1), end);
  const bool writes_units = blockIdx.x == 0 && blockIdx.y == 0;
  if (writes_units && tid == 0) {
    p.units[p.r.n_seq] = line.each;
    p.units[p.r.n_seq + 1] = line.more;
  }
  if (u0 >= u1) return;

  int carry = 0;
  for (; c0 < p.r.n_seq && (writes_units || carry < u1); c0 += kAttendThreads) {
    if (p.r.n_seq > kAttendThreads) {
      __syncthreads();
      take(c0);  // (one chunk's requests are there)
    }
    v[0] = line.weight(own.units);
    block_scan<kAttendThreads, 1>(v, all, s_sum);
    if (writes_units && c0 + tid < p.r.n_seq) p.units[c0 + tid] = carry + v[0];
    const int to = min(u1, carry + all[0] - max(line.start, 0));  // (what a chunk's last request takes more is no group)
    for (int at = max(u0, carry); at < to;) {
      // the request that `at` lies in, or the one behind the gap that it lies in: one thread's
      const int unit = at - carry - v[0], before = line.start < 0 || v[0] == 0 ? 0 : line.start;
      if (own.units > 0 && unit < own.units && unit >= -before) {
        s_seen = own;
        s_at[0] = tid;
        s_at[1] = v[0];
      } else if (line.start < 0 && own.units > 0 && unit >= own.units && unit < line.weight(own.units)) {
        s_at[0] = -1;  // (behind a request's groups: the piece is done)
      }
      lds_barrier();
      const int request = uniform(s_at[0]);
      if (request < 0) break;
      const Seen s = {uniform(s_seen.tokens), uniform(s_seen.row),    uniform(s_seen.queries),
                      uniform(s_seen.first),  uniform(s_seen.groups), uniform(s_seen.units)};
      const int i = c0 + request;
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

      attend4_share<D, NT, ONCE, kAttendWaves>(
          p, s, i, g0, g1, h, vector0, vectors, begin >= u0 && end <= u1,
          p.partial + (((int64_t)blockIdx.y * p.parts + blockIdx.x) * 2 + (begin <= u0 ? 0 : 1)) * (kVectors * (D + 2)));
    }
    carry += all[0];
  }
}

// One workgroup for each request, and nothing to join.
template <int D, int NT, bool ONCE, int WAVES>
__global__ __launch_bounds__(64 * WAVES, WAVES > kAttendWaves ? 2 : attend4_waves(D, NT))
    void attend4_whole_kernel(const AttendParams p) {
  const int heads = p.c.kv_heads, h = blockIdx.y % heads, vector0 = (blockIdx.y / heads) * 16 * NT;
  const Seen s = seen_of(p, blockIdx.x);
  const int vectors = (int)min<int64_t>((int64_t)min(s.queries, p.max_q) * p.group - vector0, 16 * NT);
  if (vectors > 0)
    attend4_share<D, NT, ONCE, WAVES>(p, s, blockIdx.x, s.first, s.first + s.groups, h, vector0, vectors, true, nullptr);
  fill_past<D>(p, s, blockIdx.y, threadIdx.x, 64 * WAVES);
}

// Joins a request's shares: O = sum of 2^(m_w - M) O_w over sum of 2^(m_w - M) l_w, in an order that the sizes alone set.
// Requests that one workgroup took whole are done already. Up to kFew shares: a thread walks them for four elements of a
// vector. More: 64 elements of a vector by 16 threads of four and 16 rows, each row with every sixteenth share, and the rows
// joined through LDS. A launch and three rounds of dependent loads bound it: 48 requests, 32 heads of 128, 4.1 us; one request
// over 256 shares, 32 heads of 512, 4.7.
template <int D>
__global__ __launch_bounds__(256) void join4_kernel(const AttendParams p, int vectors_per) {
  constexpr int kSlabs = D / 64, kFew = 4;
  __shared__ float s_m[16], s_l[16];
  __shared__ f32x4 s_x[16][16];
  const int i = blockIdx.x, heads = p.c.kv_heads;
  const Line line = {p.units[p.r.n_seq], p.units[p.r.n_seq + 1], 0};
  const int begin = p.units[i];
  const Seen s = seen_of(p, i);
  if (s.units == 0) return;
  fill_past<D>(p, s, blockIdx.y, blockIdx.z * 256 + threadIdx.x, gridDim.z * 256);
  const int first = line.part_of(begin), last = line.part_of(begin + s.units - 1);
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
    const float* const part = base + (2 * (int64_t)w + (w == first && begin > line.begin(w) ? 1 : 0)) * size;
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
  const dim3 grid(x, y), threads(kAttendThreads);
  if (p.whole) {
    if constexpr (NT == 1 && D <= 256) {
      if (s.wide) {
        attend4_whole_kernel<D, NT, true, 2 * kAttendWaves><<<grid, dim3(2 * kAttendThreads), 0, stream>>>(p);
        return;
      }
    }
    if (s.tiles == 1)
      attend4_whole_kernel<D, NT, true, kAttendWaves><<<grid, threads, 0, stream>>>(p);
    else
      attend4_whole_kernel<D, NT, false, kAttendWaves><<<grid, threads, 0, stream>>>(p);
    return;
  }
  if (s.tiles == 1) attend4_kernel<D, NT, true><<<grid, threads, 0, stream>>>(p);
  else attend4_kernel<D, NT, false><<<grid, threads, 0, stream>>>(p);
  // a workgroup for 64 elements of each vector, or as many as fill the GPU several times over
  const int64_t pairs = (int64_t)p.r.n_seq * y, most = (2048 + pairs - 1) / pairs, items = (int64_t)s.used * (D / 64);
  const unsigned z = (unsigned)(items < most ? items : most);
  join4_kernel<D><<<dim3((unsigned)p.r.n_seq, y, z), dim3(256), 0, stream>>>(p, 16 * NT);
}

}  // namespace

AttendShape attend4_shape(const CacheRef& c, int32_t n_seq, int32_t group, int32_t max_q, int64_t seen) {
  AttendShape s;
  const int64_t vectors = (int64_t)max_q * group;
  const int most = c.head_dim <= 128 ? 4 : c.head_dim == 256 ? 2 : 1;  // tiles of 16 vectors that the registers hold
  const int tiles = vectors <= 16 || most == 1 ? 1 : vectors <= 32 || most == 2 ? 2 : 4;
  s.vectors = 16 * tiles;
  s.tiles = (int)((vectors + s.vectors - 1) / s.vectors);
  if (s.tiles < 1) s.tiles = 1;
  const int64_t y = (int64_t)c.kv_heads * s.tiles;
  const int64_t parts = 256 * attend4_waves(c.head_dim, tiles) / y;
  s.parts = parts < 1 ? 1 : (int)parts;
  s.used = (int)(vectors < s.vectors ? vectors : s.vectors);
  s.whole = seen <= (n_seq * y > 128 ? most_whole_tokens4(c.head_dim) : whole_tokens4(c.head_dim));
  // Twice the waves where a CU has one workgroup at most and its four waves would have more than two groups each. us with four,
  // with eight, at heads of 128 with 16 key heads: 8 requests of 60 tokens 7.3, 7.8, of 250 8.4, 8.7, of 640 11.5, 10.3; 16 of 1,000
  // 15.7, 13.5; 32 (512 workgroups) of 250 10.4, 11.3, of 640 15.3, 15.1; 8 heads of 256, 32 requests of 1,000 21.5, 19.5.
  s.wide = s.whole && tiles == 1 && s.tiles == 1 && c.head_dim <= 256 && n_seq * y <= 256 && seen > 256;
  s.units_bytes = (4 * ((int64_t)n_seq + 2) + 255) / 256 * 256;
  s.bytes = s.whole ? 0 : s.units_bytes + y * s.parts * 2 * s.vectors * (c.head_dim + 2) * 4;
  return s;
}

hipError_t launch_cache4_attend(const AttendParams& p, const AttendShape& s, hipStream_t stream) {
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
