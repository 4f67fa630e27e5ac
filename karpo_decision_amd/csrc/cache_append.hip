// The block cache's append with the norms and the position rotation on the way (karpo_cache_append_rope), and every append of
// the cache in 4 bits (karpo_cache4_append).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "cache.h"
#include "cache_common.h"
#include "karpo_cache.h"
#include "karpo_cache4.h"

namespace karpo {

namespace {

typedef short s16x2 __attribute__((ext_vector_type(2)));

// x's sum / maximum over N neighbouring lanes (N = 4, 8, .. 64; in every one of them).
template <int N, class F>
__device__ __forceinline__ unsigned over_lanes(unsigned x, F join) {
  x = join(x, (unsigned)__builtin_amdgcn_update_dpp(0, x, 0xb1, 0xf, 0xf, true));  // quad_perm 1 0 3 2
  x = join(x, (unsigned)__builtin_amdgcn_update_dpp(0, x, 0x4e, 0xf, 0xf, true));  // quad_perm 2 3 0 1
  if constexpr (N >= 8) x = join(x, (unsigned)__builtin_amdgcn_update_dpp(0, x, 0x141, 0xf, 0xf, true));   // mirrored within 8
  if constexpr (N >= 16) x = join(x, (unsigned)__builtin_amdgcn_update_dpp(0, x, 0x140, 0xf, 0xf, true));  // within 16
  if constexpr (N >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = join(r[0], r[1]);
  }
  if constexpr (N >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    x = join(r[0], r[1]);
  }
  return x;
}
template <int N>
__device__ __forceinline__ float sum_over(float x) {
  return __uint_as_float(over_lanes<N>(__float_as_uint(x), [](unsigned a, unsigned b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}
template <int N>
__device__ __forceinline__ unsigned max_over(unsigned x) {
  return over_lanes<N>(x, [](unsigned a, unsigned b) { return max(a, b); });
}

// 1 / sqrt(x), less than a step off: the instruction's estimate and one Newton step. (The instruction takes no subnormal numbers:
// they are scaled first; 0 gives infinity, infinity 0.)
__device__ __forceinline__ float reciprocal_root(float x) {
  const bool small = x < 0x1p-96f;
  x = small ? x * 0x1p64f : x;
  const float v = __builtin_amdgcn_rsqf(x), e = __builtin_fmaf(-x * v, v, 1.f);
  const float r = e == e ? __builtin_fmaf(0.5f * v, e, v) : v;
  return small ? r * 0x1p32f : r;
}

// The least e with m <= 448 * 2^e (448 = 1.75 * 2^8), with BITS 4 m <= 6 * 2^e (6 = 1.5 * 2^2), for the fp32 magnitude with
// these bits.
template <int BITS>
__device__ __forceinline__ int exponent_of(unsigned bits) {
  const int e = (int)(bits >> 23) - 127;
  if constexpr (BITS == 8)
    return min(max(e - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0), KARPO_CACHE_MIN_EXP), KARPO_CACHE_MAX_EXP);
  else
    return min(max(e - 2 + ((bits & 0x7fffff) > 0x400000 ? 1 : 0), KARPO_CACHE4_MIN_EXP), KARPO_CACHE4_MAX_EXP);
}

// Four fp32 over `scale` as e4m3 codes, eight as e2m1 codes (nearest, ties to even).
__device__ __forceinline__ unsigned codes8(float a, float b, float c, float d, float scale) {
  const s16x2 low = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(s16x2{0, 0}, a, b, scale, false);
  return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(low, c, d, scale, true));
}
__device__ __forceinline__ unsigned codes4(const float (&y)[8], float scale) {
  unsigned w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0, y[0], y[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[2], y[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[4], y[5], scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[6], y[7], scale, 3);
}
// Four e4m3 codes under the scale `old` as codes under `scale`: rounded again.
__device__ __forceinline__ unsigned codes_again(unsigned w, float old, float scale) {
  auto at = [](unsigned pair, bool up) { return __uint_as_float(up ? pair & 0xffff0000u : pair << 16); };
  const unsigned a = bf16_pair(w, old, false), b = bf16_pair(w, old, true);
  return codes8(at(a, false), at(a, true), at(b, false), at(b, true), scale);
}

// A write: `count` tokens from slot `first` of a block on, out of the rows from `row` on.
struct Write {
  int block, first, row, count;
};

// One write's keys, or values, of one head: WAVES waves, D / 8 lanes a token of 8 elements each (16 bytes a lane and load), the
// tokens in PASSES passes. y = x * rsqrt(mean x^2 + eps) * w, its first rope_dim elements turned by halves, in fp32; the one
// rounding is that to the codes. A token's sum of squares and, in 4 bits, the largest of 32 elements (four lanes) go across
// lanes in registers; the element half a rotation away comes from its lane as the raw bf16 pair, normed again here. In 8 bits all
// rows stay in registers until the block's maximum is known. Keys are stored from there (a token's 64 elements lie together);
// of values the tokens lie innermost, so their codes go through LDS, a token's side by side, out of which a lane takes 4 tokens x
// 4 bytes four times: four 16-byte pieces of the cache. Lanes past the write take its last token again and store nothing, so
// that loads need no branches and all passes' are in flight at once.
//
// Many rows are bound by HBM: 32,768 of 16 heads of 128, normed and rotated, 90 us in 8 bits (402 MB and 17 MB of tables, 4.7 TB/s;
// 145 with loads pass by pass and one head a workgroup) and 78 us in 4 (356 MB); few by three rounds of dependent loads (the write,
// its rows and positions, cos and sin) and the joins over the workgroup: one token of 48 requests 6.7 us, 2,500 tokens of 24
// requests, 8 heads of 256, 14.4. Of four such documents' 537 million codes 278 are another than the 64-bit rows' (566 where each
// step of the formulas is rounded to fp32 by itself): elements that close to the border between two codes. With the root as a
// sum of two terms 273, and 93.5 us.
template <int D, int BLOCK, int PASSES, int WAVES, int BITS, bool MANY, bool VALUE, bool TURNED>
__device__ __forceinline__ void append_rows(const AppendRowsParams& p, const Write& wr, int h0, int h1, char* s_codes) {
  constexpr int kLanes = D / 8, kRows = 64 / kLanes, kStep = kRows * WAVES;
  constexpr int kBytes = BITS == 8 ? D : D / 2;  // of a token's codes
  constexpr int kPitch = kBytes + 16;
  const CacheRef& c = p.a.c;
  const int first = wr.first, count = wr.count;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int sub = lane / kLanes, l = lane - sub * kLanes, d0 = l * 8;
  const int64_t stride = VALUE ? p.a.sv_t : p.a.sk_t;
  const uint16_t* const in = (VALUE ? p.a.v : p.a.k) + wr.row * stride + d0;
  auto token_of = [&](int t) { return t * kStep + wave * kRows + sub; };

  // norm: (x * w) * r, w the weight, 1 + weight or 1; rotation of the first rope_dim elements, partner rh away. A product of two
  // bf16 numbers, and of three, is exact in fp32, so a weighted key takes two roundings, (xw * cos - xw' * sin) and the
  // product with r (normed first and then turned it is five; where w is 1 + weight, that sum and its products round too).
  const NormRef& norm = VALUE ? p.v_norm : p.k_norm;
  const bool normed = norm.mode != KARPO_NORM_NONE;
  const float wm = norm.mode == KARPO_NORM_WEIGHT || norm.mode == KARPO_NORM_ONE_PLUS ? 1.f : 0.f;
  const float wa = norm.mode == KARPO_NORM_WEIGHT ? 0.f : 1.f;
  const int rd = TURNED ? p.rope_dim : 0, rh = rd >> 1;
  const bool inside = d0 < rd;
  const int dp = inside ? (d0 < rh ? d0 + rh : d0 - rh) : d0;

  // the tokens' rows of the tables, for all heads; the first head's rows; the norm's weight (a next head's rows are loaded when the
  // last one's are through)
  int64_t at[PASSES];
  if constexpr (TURNED) {
#pragma unroll
    for (int t = 0; t < PASSES; ++t) {
      at[t] = (int64_t)wr.row + min(token_of(t), count - 1);
      if (p.positions != nullptr) at[t] = p.positions[at[t]];
    }
  }
  u32x4 x[PASSES], cv[PASSES], sv[PASSES];
  auto load = [&](int h) {  // head h's rows
#pragma unroll
    for (int t = 0; t < PASSES; ++t) {
      const u32x4* const from = reinterpret_cast<const u32x4*>(in + min(token_of(t), count - 1) * stride +
                                                               h * (VALUE ? p.a.sv_h : p.a.sk_h));
      if constexpr (MANY) x[t] = __builtin_nontemporal_load(from); else x[t] = *from;
    }
  };
  load(h0);
  u32x4 wv = {0, 0, 0, 0}, wp = {0, 0, 0, 0};
  if (wm != 0.f) {
    wv = *reinterpret_cast<const u32x4*>(norm.weight + d0);
    if constexpr (TURNED) wp = *reinterpret_cast<const u32x4*>(norm.weight + dp);
  }
  if constexpr (TURNED) {
#pragma unroll
    for (int t = 0; t < PASSES; ++t) {
      const bool known = at[t] >= 0 && at[t] < p.rope_rows;
      const int64_t from = (known ? at[t] : 0) * p.rope_stride + (inside ? d0 : 0);
      cv[t] = *reinterpret_cast<const u32x4*>(p.cos + from);
      sv[t] = *reinterpret_cast<const u32x4*>(p.sin + from);
      if (!known) cv[t] = u32x4{kNanPair, kNanPair, kNanPair, kNanPair};
    }
  }
  float w_mine[8], w_other[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    w_mine[e] = wm * bf16_at(wv, e) + wa;
    w_other[e] = (wm * bf16_at(wp, e) + wa) * (d0 < rh ? -1.f : 1.f);
  }
  const int partner = (sub * kLanes + (dp >> 3)) * 4;  // its lane's byte address

  int h = h0;
  do {
    if constexpr (MANY && TURNED) {  // (kept as they are: their 64 elements in fp32 would be registers over all heads)
#pragma unroll
      for (int t = 0; t < PASSES; ++t)
#pragma unroll
        for (int k = 0; k < 4; ++k) asm volatile("" : "+v"(cv[t][k]), "+v"(sv[t][k]));
    }
    const int64_t head = (int64_t)wr.block * c.kv_heads + h;
    uint8_t* const out = (VALUE ? c.values : c.keys) + head * BLOCK * kBytes;
    float* const scale_of = BITS == 8 ? c.scales + 2 * head + (VALUE ? 1 : 0) : nullptr;
    const unsigned old_bits = BITS == 8 && first > 0 ? __float_as_uint(*scale_of) : 0;
    auto row_of = [&](int t, float (&y)[8]) {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(bf16_at(x[t], e), bf16_at(x[t], e), ss);
      const float root = reciprocal_root(sum_over<kLanes>(ss) * (1.f / D) + norm.eps), r = normed ? root : 1.f;
      if constexpr (TURNED) {
        u32x4 px;
#pragma unroll
        for (int k = 0; k < 4; ++k) px[k] = (unsigned)__builtin_amdgcn_ds_bpermute(partner, (int)x[t][k]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float n = bf16_at(x[t], e) * w_mine[e];
          const float turn = __builtin_fmaf(n, bf16_at(cv[t], e), bf16_at(px, e) * w_other[e] * bf16_at(sv[t], e));
          y[e] = (inside ? turn : n) * r;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = bf16_at(x[t], e) * w_mine[e] * r;
      }
    };
    // the largest magnitude of y and `best`, NaN as nothing
    auto larger = [&](const float (&y)[8], float best) {
#pragma unroll
      for (int e = 0; e < 8; e += 2)
        best = __builtin_fmaxf(__builtin_fmaxf(best, __builtin_fabsf(y[e])), __builtin_fabsf(y[e + 1]));
      return best;
    };

    bool grown = false;
    float scale = 1.f, old_scale = 1.f;
    if constexpr (BITS == 8) {
      float y[PASSES][8], most_of = 0.f;
#pragma unroll
      for (int t = 0; t < PASSES; ++t) {
        row_of(t, y[t]);
        most_of = larger(y[t], most_of);
      }
      if (MANY && h + 1 < h1) load(h + 1);
      auto joined = [&](unsigned mine) {  // over the workgroup
        mine = max_over<64>(mine);
        if constexpr (WAVES > 1) {
          unsigned* const s_best = reinterpret_cast<unsigned*>(s_codes);
          __syncthreads();
          if (lane == 0) s_best[wave] = mine;
          __syncthreads();
#pragma unroll
          for (int w = 0; w < WAVES; ++w) mine = max(mine, s_best[w]);
          __syncthreads();  // (the codes, or the next head's maxima, take the array)
        }
        return mine;
      };
      unsigned best = joined(__float_as_uint(most_of));
      const bool odd = best >= 0x7f800000u;  // infinities: the largest of the others
      if (__builtin_expect(odd, 0)) {
        best = 0;
#pragma unroll
        for (int t = 0; t < PASSES; ++t)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const unsigned m = __float_as_uint(y[t][e]) & 0x7fffffffu;
            best = max(best, m < 0x7f800000u ? m : 0u);
          }
        best = joined(best);
      }
      int e = exponent_of<8>(best), old = e;
      if (first > 0) {
        old = min(max((int)((old_bits >> 23) & 0xff) - 127, KARPO_CACHE_MIN_EXP), KARPO_CACHE_MAX_EXP);
        e = max(e, old);
      }
      grown = old < e;  // the earlier tokens' codes are rounded again
      scale = power_of_two(e);
      old_scale = power_of_two(old);
      if (tid == 0) *scale_of = scale;
      if (__builtin_expect(odd || e == KARPO_CACHE_MAX_EXP, 0)) {
        const float most = 448.f * scale;
#pragma unroll
        for (int t = 0; t < PASSES; ++t)
#pragma unroll
          for (int k = 0; k < 8; ++k) y[t][k] = __builtin_fabsf(y[t][k]) > most ? __builtin_copysignf(most, y[t][k]) : y[t][k];
      }
#pragma unroll
      for (int t = 0; t < PASSES; ++t) {
        const int slot = first + token_of(t);
        const u32x2 w = {codes8(y[t][0], y[t][1], y[t][2], y[t][3], scale), codes8(y[t][4], y[t][5], y[t][6], y[t][7], scale)};
        if (token_of(t) < count) {
          if constexpr (VALUE)
            *reinterpret_cast<u32x2*>(s_codes + slot * kPitch + d0) = w;
          else
            *reinterpret_cast<u32x2*>(out + ((slot >> 4) * (D / 64) + (d0 >> 6)) * 1024 + (slot & 15) * 64 + (d0 & 63)) = w;
        }
      }
      if (!VALUE && grown) {
        for (int u = tid; u < first * (D / 16); u += 64 * WAVES) {
          const int slot = u / (D / 16), piece = u % (D / 16);
          u32x4* const dst =
              reinterpret_cast<u32x4*>(out + ((slot >> 4) * (D / 64) + (piece >> 2)) * 1024 + (slot & 15) * 64 + (piece & 3) * 16);
          u32x4 w = *dst;
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] = codes_again(w[k], old_scale, scale);
          *dst = w;
        }
      }
    } else {
      uint8_t* const scales = c.scales4 + head * (BLOCK / 32) * 2 * D + (VALUE ? D : 0);
#pragma unroll
      for (int t = 0; t < PASSES; ++t) {
        const int slot = first + token_of(t);
        float y[8];
        row_of(t, y);
        // (a sum is NaN where an element is, or where infinities of both signs are)
        unsigned best = max_over<4>(__float_as_uint(larger(y, 0.f)));
        const float sum = ((y[0] + y[1]) + (y[2] + y[3])) + ((y[4] + y[5]) + (y[6] + y[7]));
        bool nan = false;
        // seldom: the largest of the others, and is one NaN
        if (__any(!(__builtin_fabsf(sum) < INFINITY) || best >= 0x7f800000u)) {
          unsigned fine = 0, all = 0;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const unsigned m = __float_as_uint(y[e]) & 0x7fffffffu;
            fine = max(fine, m < 0x7f800000u ? m : 0u);
            all = max(all, m);
          }
          best = max_over<4>(fine);
          nan = max_over<4>(all) > 0x7f800000u;
        }
        const int e = exponent_of<4>(best);
        const unsigned w = codes4(y, power_of_two(e));
        if (token_of(t) < count) {
          const int group = d0 >> 5, t2 = (slot >> 4) & 1, t16 = slot & 15;
          if constexpr (VALUE)
            *reinterpret_cast<unsigned*>(s_codes + slot * kPitch + (d0 >> 1)) = w;
          else
            *reinterpret_cast<unsigned*>(out + (slot >> 5) * 16 * D + (t2 * (D / 32) + group) * 256 + t16 * 16 +
                                         ((d0 & 31) >> 1)) = w;
          if ((l & 3) == 0) {
            const int byte = VALUE     ? group * 32 + (t16 >> 2) * 8 + t2 * 4 + (t16 & 3)
                             : D == 64 ? (t2 * 2 + group) * 16 + t16
                                       : ((group & 3) * 16 + t16) * (D / 64) + (group >> 2) * 2 + t2;
            scales[(slot >> 5) * 2 * D + byte] = nan ? 255 : (uint8_t)(e + 127);
          }
        }
      }
      if (MANY && h + 1 < h1) load(h + 1);
    }
    if constexpr (VALUE) {
      __syncthreads();
      const int half0 = grown ? 0 : first >> 5, half1 = (first + count - 1) >> 5;
      constexpr int kTiles = kBytes / 32;  // KiB of codes of 32 tokens
      for (int u = tid; u < (half1 - half0 + 1) * kTiles * 16; u += 64 * WAVES) {
        const int j = u & 3, q = (u >> 2) & 3, tile = (u >> 4) % kTiles, half = half0 + (u >> 4) / kTiles;
        // bytes of the tokens 16 t + 4 q + 0 .. 3 that are new, and that are rounded again
        unsigned is_new[2] = {0, 0}, is_old[2] = {0, 0};
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int slot = half * 32 + t * 16 + q * 4 + i;
            if (slot >= first && slot < first + count) is_new[t] |= 0xffu << (8 * i);
            if (grown && slot < first) is_old[t] |= 0xffu << (8 * i);
          }
        if ((is_new[0] | is_new[1] | is_old[0] | is_old[1]) == 0) continue;
        const bool whole = (is_new[0] & is_new[1]) == 0xffffffffu;
        u32x4 w[4];
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            unsigned r[4], o[4];
            const char* const from = s_codes + (half * 32 + t * 16 + q * 4) * kPitch + tile * 32 + g * 16 + j * 4;
#pragma unroll
            for (int i = 0; i < 4; ++i) r[i] = *reinterpret_cast<const unsigned*>(from + i * kPitch);
            transposed(r, o);
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k][2 * g + t] = o[k];
          }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int dl = 4 * j + k;
          u32x4* const dst = reinterpret_cast<u32x4*>(out + (half * kTiles + tile) * 1024 +
                                                      (BITS == 8 ? dl * 64 + q * 16 : (q * 16 + dl) * 16));
          if (!whole) {
            const u32x4 was = *dst;
#pragma unroll
            for (int m = 0; m < 4; ++m) {
              unsigned kept = was[m];
              if constexpr (BITS == 8)
                if (grown) kept = (codes_again(kept, old_scale, scale) & is_old[m & 1]) | (kept & ~is_old[m & 1]);
              w[k][m] = (w[k][m] & is_new[m & 1]) | (kept & ~is_new[m & 1]);
            }
          }
          *dst = w[k];
        }
      }
      if (MANY && h + 1 < h1) __syncthreads();  // (the next head's codes take the array)
    }
  } while (MANY && ++h < h1);
}

// (three waves a SIMD where one walks heads over 8 bits: without the bound two, and a document of 16 heads of 128 93.8 us, not
// 89.6. Otherwise as the registers have it: 89 to 93 of them in 4 bits and 106 to 121 in 8, 133 and so three waves in blocks of 32
// at heads of 64 and 512. Sixteen waves at heads of 512 have 128 each and spill: in blocks of 128 5 in 4 bits and 7 in 8, in
// blocks of 64 1 in 8.)
template <int D, int BLOCK, int PASSES, int WAVES, int BITS, bool MANY>
__global__ __launch_bounds__(64 * WAVES, MANY && BITS == 8 ? 3 : 1) void append_rows_kernel(const AppendRowsParams p) {
  constexpr int kStep = 512 / D * WAVES;  // tokens of a pass
  __shared__ __align__(16) char s_codes[BLOCK * ((BITS == 8 ? D : D / 2) + 16)];
  const int heads = p.a.c.kv_heads, groups = (heads + p.heads_each - 1) / p.heads_each;  // (of heads)
  const int64_t unit = blockIdx.x / (2 * groups);
  const int which = (int)(blockIdx.x - unit * 2 * groups), h0 = (which >> 1) * p.heads_each, h1 = min(h0 + p.heads_each, heads);
  const int4 w = *reinterpret_cast<const int4*>(p.a.writes + 4 * unit);
  const Write wr = {w.x, w.y, w.z, w.w};
  if (wr.count < 1 || wr.block < 0 || wr.block >= p.a.c.blocks || wr.first < 0 || wr.count > BLOCK - wr.first || wr.row < 0 ||
      wr.row > p.a.rows - wr.count)
    return;
  auto run = [&](auto passes) {
    constexpr int N = decltype(passes)::value;
    if (which & 1)
      append_rows<D, BLOCK, N, WAVES, BITS, MANY, true, false>(p, wr, h0, h1, s_codes);
    else if (p.cos != nullptr)
      append_rows<D, BLOCK, N, WAVES, BITS, MANY, false, true>(p, wr, h0, h1, s_codes);
    else
      append_rows<D, BLOCK, N, WAVES, BITS, MANY, false, false>(p, wr, h0, h1, s_codes);
  };
  if (wr.count <= kStep) run(std::integral_constant<int, 1>()); else run(std::integral_constant<int, PASSES>());
}

// Passes of a workgroup, whose loads are all in flight at once. With 2 (twice the waves) one token of 48 requests, 16 heads of 128:
// 8.7 against 6.6 us, 2,500 tokens of 24 requests, 8 heads of 256: 19.5 against 14.3, 32,768 tokens of 16 heads of 128: 89.7
// against 93.2.
constexpr int kMostPasses = 4;

template <int D, int BITS>
hipError_t launch(const AppendRowsParams& p, hipStream_t stream) {
  auto run = [&](auto blocks) {
    constexpr int kBlock = decltype(blocks)::value, kPieces = D * kBlock / 512;  // of 64 lanes x 8 elements
    constexpr int kWaves = kPieces <= 16 * kMostPasses ? kPieces / kMostPasses : 16, kPasses = kPieces / kWaves;
    // Many rows (over 96 MiB of keys and values: as many as come from HBM): up to eight heads a workgroup, which then load their
    // tokens' cos and sin once, while there are four workgroups a CU, and the rows past the caches. us with it, without, rotated, in
    // 8 bits, 16 heads of 128: 64 MiB 29.8, 27.3; 128 MiB 52.0, 58.9; 256 MiB 84.4, 106; 8 of 256: 64 MiB 37.9, 31.5; 128 MiB 64.5,
    // 67.2; 256 MiB 104, 124; 4 of 512 in blocks of 32: 128 MiB 62.2, 94.9; in 4 bits (and read back) 16 of 128: 128 MiB 76.3, 87.2;
    // 4 of 512: 64 MiB 57.5, 53.7; 128 MiB 94.0, 99.5. Not where sixteen waves leave too few registers for it: blocks of 32 Ki
    // elements in 8 bits (8 heads of 256, blocks of 128: 128 MiB 110, 79.8; 4 of 512, blocks of 64: 112, 93.1), of 64 Ki in both.
    constexpr bool kMany = kPasses <= kMostPasses && !(BITS == 8 && kWaves == 16);
    AppendRowsParams q = p;
    q.heads_each = 1;
    const bool many = kMany && 4 * p.a.rows * p.a.c.kv_heads * D > (int64_t)96 << 20;
    while (many && q.heads_each < 8 && p.n_writes * p.a.c.kv_heads >= 1024 * q.heads_each) q.heads_each *= 2;
    const dim3 grid((unsigned)(p.n_writes * 2 * ((p.a.c.kv_heads + q.heads_each - 1) / q.heads_each)));
    if constexpr (kMany) {
      if (many) {
        append_rows_kernel<D, kBlock, kPasses, kWaves, BITS, true><<<grid, dim3(64 * kWaves), 0, stream>>>(q);
        return;
      }
    }
    append_rows_kernel<D, kBlock, kPasses, kWaves, BITS, false><<<grid, dim3(64 * kWaves), 0, stream>>>(q);
  };
  switch (p.a.c.block_log2) {
    case 5: run(std::integral_constant<int, 32>()); break;
    case 6: run(std::integral_constant<int, 64>()); break;
    case 7: run(std::integral_constant<int, 128>()); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_cache_append_rows(const AppendRowsParams& p, hipStream_t stream) {
  const bool four = p.a.c.scales4 != nullptr;
  switch (p.a.c.head_dim) {
    case 64: return four ? launch<64, 4>(p, stream) : launch<64, 8>(p, stream);
    case 128: return four ? launch<128, 4>(p, stream) : launch<128, 8>(p, stream);
    case 256: return four ? launch<256, 4>(p, stream) : launch<256, 8>(p, stream);
    case 512: return four ? launch<512, 4>(p, stream) : launch<512, 8>(p, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace karpo
