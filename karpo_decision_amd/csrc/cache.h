// The block cache's kernels' arguments (cache.hip, cache_append.hip, cache_attn.hip, cache4_attn.hip), shared with the C ABI
// (cache_capi.cpp).
#pragma once
#include <hip/hip_runtime_api.h>
#include <stdint.h>

namespace karpo {

constexpr int kCacheGroup = 32;  // tokens that a wave takes at once: two key tiles, one row of value tiles

struct CacheRef {
  uint8_t* keys;
  uint8_t* values;
  float* scales;     // of a cache in 8 bits, null otherwise
  uint8_t* scales4;  // of a cache in 4 bits, null otherwise
  int64_t blocks;
  int32_t kv_heads, head_dim, block_log2;
};

// A batch's cached tokens: request i's lie in the blocks table[i * table_stride + ..], lengths[i] of them, at most
// `most` (the table row's).
struct CacheRows {
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lengths;
  int32_t n_seq, most;
};

struct ReserveParams {
  int32_t* table;
  int64_t table_stride;
  int64_t most;  // tokens a table row holds
  const int32_t* lengths;
  const int32_t* counts;
  const int32_t* free_blocks;
  const int32_t* free_count;
  int32_t* q_cu;
  int32_t* new_lengths;
  int64_t* slots;
  int32_t* positions;
  int32_t* writes;
  int32_t* free_left;
  int32_t* status;
  int32_t n_seq, free_capacity, block_log2;
  int32_t rows, per, writes_capacity;  // per: rows of each workgroup (set by the launch)
};
hipError_t launch_cache_reserve(ReserveParams p, hipStream_t stream);

struct AppendParams {
  CacheRef c;
  const uint16_t* k;
  const uint16_t* v;
  int64_t sk_t, sk_h, sv_t, sv_h;
  const int32_t* writes;
  int64_t rows;
};
hipError_t launch_cache_append(const AppendParams& p, int64_t n_writes, hipStream_t stream);

// `append` with norms and rotation, and every `append` of a cache in 4 bits.
struct NormRef {
  int32_t mode;  // KARPO_NORM_*
  float eps;
  const uint16_t* weight;  // or null
};
struct AppendRowsParams {
  AppendParams a;
  NormRef k_norm, v_norm;
  const uint16_t* cos;  // or null: no rotation
  const uint16_t* sin;
  int64_t rope_stride, rope_rows;
  int32_t rope_dim;
  const int32_t* positions;  // each row's row of the tables, or null: its own
  int64_t n_writes;
  int32_t heads_each;  // heads that a workgroup takes, one after the other (the launch's)
};
hipError_t launch_cache_append_rows(const AppendRowsParams& p, hipStream_t stream);

struct ReadParams {
  CacheRef c;
  CacheRows r;
  const int32_t* q_cu;  // with it: only the tokens that a request's queries can see (window_left before the first)
  int32_t window_left;
  // with q_cu, where bounds do not hold (query rows past total_q or out of order, more than max_q of them, more tokens than
  // `rows`): the packed attention behind this computes nothing then, and all requests' rows of o become NaN
  int32_t max_q;
  int64_t total_q;
  uint16_t* o;
  int64_t so_t, so_h;
  int32_t heads;
  int32_t no_scale;  // the scale is NaN, and nothing runs behind this: NaN as well, zeros for requests without tokens
  uint16_t* k;
  uint16_t* v;
  int64_t rows;
  int32_t* k_cu;
  int32_t stream;  // the rows are more than the L2 caches hold: stored through them
};
hipError_t launch_cache_read(const ReadParams& p, hipStream_t stream);

struct AttendParams {
  CacheRef c;
  CacheRows r;
  const uint16_t* q;
  uint16_t* o;
  int64_t sq_t, sq_h, so_t, so_h;
  const int32_t* q_cu;
  int64_t total_q;
  int32_t max_q;       // rows of a request's queries behind this many become NaN
  int32_t group;       // heads / kv_heads
  float per_group;     // 1 / group
  int32_t whole;       // a workgroup takes a request whole (nothing to join)
  int32_t left, right;
  float scale;         // its magnitude times log2(e), at least 1e-30 (hidden scores, -infinity, stay that)
  uint32_t sign;       // 0x80008000 where the scale is negative: the queries are
  int32_t parts;       // workgroups for each of the grid's y
  float* partial;      // [y][parts][2] of (O [vectors][D], m [vectors], l [vectors])
  int32_t* units;      // [n_seq + 1] groups of 32 tokens before each request (in 4 bits [n_seq + 2]: where each begins on the
                       // line that the workgroups cut, and the pieces)
};

// The split path's launch for these sizes: `vectors` query vectors (position x head of the group) per workgroup, `tiles`
// workgroups for a key/value head's max_q * group vectors, `parts` shares of the keys.
struct AttendShape {
  int vectors, used, tiles, parts;  // used: the most of them that any workgroup has
  bool whole;
  int64_t units_bytes, bytes;  // of the workspace: the units, then the partials
  bool wide = false;  // whole, in 4 bits: by eight waves a request
};
// `seen`: a bound of the tokens that a request's queries see.
AttendShape attend_shape(const CacheRef& c, int32_t n_seq, int32_t group, int32_t max_q, int64_t seen);
hipError_t launch_cache_attend(const AttendParams& p, const AttendShape& s, hipStream_t stream);
// The same for a cache in 4 bits.
AttendShape attend4_shape(const CacheRef& c, int32_t n_seq, int32_t group, int32_t max_q, int64_t seen);
hipError_t launch_cache4_attend(const AttendParams& p, const AttendShape& s, hipStream_t stream);

}  // namespace karpo
