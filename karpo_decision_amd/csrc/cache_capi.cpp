// The block cache's C ABI (karpo_cache.h): argument checks, workspace sizes and launches. Everything that the kernels
// index with is checked here or in the kernel itself, before a launch or a load.
#include <math.h>
#include <stdint.h>
#include <string.h>

#include "cache.h"
#include "karpo_cache.h"

using namespace karpo;

namespace {

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int block_log2(int32_t block_size) { return block_size == 32 ? 5 : block_size == 64 ? 6 : block_size == 128 ? 7 : -1; }

bool overlaps(const void* a, int64_t na, const void* b, int64_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return na > 0 && nb > 0 && x < y + (uintptr_t)nb && y < x + (uintptr_t)na;
}

// Tokens of a table's row; all rows of a table in groups of 32 tokens (and 64 more each, which the shares add) fit 32 bits.
constexpr int64_t kMostTokens = (int64_t)1 << 26;

int check_cache(const KarpoCache& c, CacheRef* ref) {
  const int b = block_log2(c.block_size);
  if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256 && c.head_dim != 512) return KARPO_ATTN_ERR_HEAD_DIM;
  if (c.kv_heads < 1 || c.kv_heads > 8192) return KARPO_ATTN_ERR_HEADS;
  if (b < 0 || c.blocks < 1 || c.blocks > INT32_MAX) return KARPO_ATTN_ERR_ARG;
  if (!c.keys || !c.values || !c.scales) return KARPO_ATTN_ERR_NULL;
  if (!aligned(c.keys, 16) || !aligned(c.values, 16) || !aligned(c.scales, 8)) return KARPO_ATTN_ERR_LAYOUT;
  ref->keys = static_cast<uint8_t*>(c.keys);
  ref->values = static_cast<uint8_t*>(c.values);
  ref->scales = c.scales;
  ref->blocks = c.blocks;
  ref->kv_heads = c.kv_heads;
  ref->head_dim = c.head_dim;
  ref->block_log2 = b;
  return KARPO_ATTN_OK;
}

int check_rows(const int32_t* table, int64_t stride, int32_t width, const int32_t* lengths, int32_t n_seq,
               int32_t block_size, CacheRows* rows) {
  if (n_seq < 0 || width < 1 || stride < width || (int64_t)width * block_size > kMostTokens) return KARPO_ATTN_ERR_ARG;
  if ((int64_t)n_seq * ((int64_t)width * block_size / kCacheGroup + 64) > INT32_MAX) return KARPO_ATTN_ERR_ARG;
  if (n_seq > 0 && (!table || !lengths)) return KARPO_ATTN_ERR_NULL;
  rows->table = table;
  rows->table_stride = stride;
  rows->lengths = lengths;
  rows->n_seq = n_seq;
  rows->most = (int32_t)(width * (int64_t)block_size);
  return KARPO_ATTN_OK;
}

// The eight L2 caches. Rows past them are stored through: 32,768 of 16 heads at 128 77.9 -> 71.4 us, six requests at head size
// 512 (75 MB) 22.5 -> 20.0; the attention's own unpacked rows are read next and are not (chunks over 30,000 tokens: equal).
constexpr int64_t kL2Bytes = (int64_t)32 << 20;

bool row_strides(const void* p, int64_t tok, int64_t head) {
  return aligned(p, 16) && tok >= 0 && head >= 0 && tok % 8 == 0 && head % 8 == 0;
}

}  // namespace

extern "C" int64_t karpo_cache_writes_capacity(int64_t rows, int32_t n_seq, int32_t block_size) {
  const int b = block_log2(block_size);
  if (rows < 0 || rows > INT32_MAX || n_seq < 0 || b < 0) return 0;
  // a request's c > 0 tokens touch at most min(c, c / block_size + 2) blocks
  const int64_t blocks = (rows >> b) + 2 * (int64_t)n_seq;
  return rows < blocks ? rows : blocks;
}

extern "C" int karpo_cache_reserve(const KarpoCacheReserveArgs* a, void* stream) {
  if (a == nullptr) return KARPO_ATTN_ERR_NULL;
  const int b = block_log2(a->block_size);
  if (b < 0 || a->rows < 0 || a->rows > INT32_MAX - 65536 || a->free_capacity < 0 ||
      a->writes_capacity != karpo_cache_writes_capacity(a->rows, a->n_seq, a->block_size))
    return KARPO_ATTN_ERR_ARG;
  CacheRows rows;
  const int st = check_rows(a->table, a->table_stride, a->width, a->lengths, a->n_seq, a->block_size, &rows);
  if (st != KARPO_ATTN_OK) return st;
  const int64_t n = a->n_seq;
  if ((n > 0 && (!a->counts || !a->new_lengths)) || (a->free_capacity > 0 && !a->free_blocks) || !a->free_count ||
      !a->q_cu || !a->free_left || !a->status ||
      (a->rows > 0 && (!a->slots || !a->positions)) || (a->writes_capacity > 0 && !a->writes))
    return KARPO_ATTN_ERR_NULL;
  if (!aligned(a->slots, 8) || !aligned(a->writes, 16)) return KARPO_ATTN_ERR_LAYOUT;
  // workgroups read the inputs while others write their outputs
  const struct { const void* p; int64_t bytes; } in[] = {
      {a->lengths, 4 * n}, {a->counts, 4 * n}, {a->free_blocks, 4 * (int64_t)a->free_capacity}, {a->free_count, 4}};
  const struct { const void* p; int64_t bytes; } out[] = {
      {a->table, n > 0 ? 4 * ((n - 1) * a->table_stride + a->width) : 0}, {a->q_cu, 4 * (n + 1)},
      {a->new_lengths, 4 * n}, {a->slots, 8 * a->rows}, {a->positions, 4 * a->rows},
      {a->writes, 16 * a->writes_capacity}, {a->free_left, 4}, {a->status, 4}};
  for (size_t i = 0; i < sizeof(out) / sizeof(out[0]); ++i) {
    for (const auto& x : in)
      if (overlaps(x.p, x.bytes, out[i].p, out[i].bytes)) return KARPO_ATTN_ERR_ARG;
    for (size_t j = 0; j < i; ++j)
      if (overlaps(out[j].p, out[j].bytes, out[i].p, out[i].bytes)) return KARPO_ATTN_ERR_ARG;
  }
  ReserveParams p;
  memset(&p, 0, sizeof(p));
  p.table = a->table;
  p.table_stride = a->table_stride;
  p.most = rows.most;
  p.lengths = a->lengths;
  p.counts = a->counts;
  p.free_blocks = a->free_blocks;
  p.free_count = a->free_count;
  p.q_cu = a->q_cu;
  p.new_lengths = a->new_lengths;
  p.slots = a->slots;
  p.positions = a->positions;
  p.writes = a->writes;
  p.free_left = a->free_left;
  p.status = a->status;
  p.n_seq = a->n_seq;
  p.free_capacity = a->free_capacity;
  p.block_log2 = b;
  p.rows = (int32_t)a->rows;
  p.writes_capacity = (int32_t)a->writes_capacity;
  if (launch_cache_reserve(p, static_cast<hipStream_t>(stream)) != hipSuccess) return KARPO_ATTN_ERR_LAUNCH;
  return KARPO_ATTN_OK;
}

extern "C" int karpo_cache_append(const KarpoCacheAppendArgs* a, void* stream) {
  if (a == nullptr) return KARPO_ATTN_ERR_NULL;
  AppendParams p;
  memset(&p, 0, sizeof(p));
  const int st = check_cache(a->cache, &p.c);
  if (st != KARPO_ATTN_OK) return st;
  if (a->rows < 0 || a->rows > INT32_MAX || a->n_writes < 0 || a->n_writes > INT32_MAX / (2 * a->cache.kv_heads))
    return KARPO_ATTN_ERR_ARG;
  const int64_t bytes = p.c.blocks * ((int64_t)p.c.kv_heads * p.c.head_dim << p.c.block_log2);
  if (overlaps(p.c.keys, bytes, p.c.values, bytes)) return KARPO_ATTN_ERR_ARG;  // (either's writes would be the other's)
  if (a->rows == 0 || a->n_writes == 0) return KARPO_ATTN_OK;
  if (!a->k || !a->v || !a->writes) return KARPO_ATTN_ERR_NULL;
  if (!row_strides(a->k, a->k_stride_tok, a->k_stride_head) || !row_strides(a->v, a->v_stride_tok, a->v_stride_head) ||
      !aligned(a->writes, 16))
    return KARPO_ATTN_ERR_LAYOUT;
  p.k = static_cast<const uint16_t*>(a->k);
  p.v = static_cast<const uint16_t*>(a->v);
  p.sk_t = a->k_stride_tok;
  p.sk_h = a->k_stride_head;
  p.sv_t = a->v_stride_tok;
  p.sv_h = a->v_stride_head;
  p.writes = a->writes;
  p.rows = a->rows;
  if (launch_cache_append(p, a->n_writes, static_cast<hipStream_t>(stream)) != hipSuccess)
    return KARPO_ATTN_ERR_LAUNCH;
  return KARPO_ATTN_OK;
}

extern "C" int karpo_cache_read(const KarpoCacheReadArgs* a, void* stream) {
  if (a == nullptr) return KARPO_ATTN_ERR_NULL;
  ReadParams p;
  memset(&p, 0, sizeof(p));
  int st = check_cache(a->cache, &p.c);
  if (st != KARPO_ATTN_OK) return st;
  st = check_rows(a->table, a->table_stride, a->width, a->lengths, a->n_seq, a->cache.block_size, &p.r);
  if (st != KARPO_ATTN_OK) return st;
  if (a->rows < 0 || a->rows > INT32_MAX) return KARPO_ATTN_ERR_ARG;
  if (!a->k_cu || (a->rows > 0 && (!a->k || !a->v))) return KARPO_ATTN_ERR_NULL;
  if (!aligned(a->k, 16) || !aligned(a->v, 16)) return KARPO_ATTN_ERR_LAYOUT;
  p.window_left = -1;
  p.k = static_cast<uint16_t*>(a->k);
  p.v = static_cast<uint16_t*>(a->v);
  p.rows = a->rows;
  p.k_cu = a->k_cu;
  p.stream = 4 * a->rows * a->cache.kv_heads * a->cache.head_dim > kL2Bytes;
  if (launch_cache_read(p, static_cast<hipStream_t>(stream)) != hipSuccess) return KARPO_ATTN_ERR_LAUNCH;
  return KARPO_ATTN_OK;
}

namespace {

int64_t round_up(int64_t x, int64_t n) { return (x + n - 1) / n * n; }

// A bound of the tokens that the queries of all requests see.
int64_t seen_keys(const KarpoCacheAttendArgs* a) {
  const int64_t each = (int64_t)a->max_q + a->window_left;
  return a->window_left >= 0 && each < a->total_keys && each * a->n_seq < a->total_keys ? each * a->n_seq : a->total_keys;
}

// The rows that the queries can see, as packed bf16 keys and values, with the packed attention's own workspace behind them.
// That kernel's weights enter its second product as one bf16 term, 2^-8 off, where the split path's are two: its matrix cores
// are what bounds it, and a second term would be half as much work again. 2-norm error against 64 bits over a chunk of 2,048 over
// 30,000 tokens 2.3e-3, of sums in fp32 (the output's rounding) 1.7e-3.
struct Unpacked {
  int64_t rows, k_offset, v_offset, ws_offset;
  size_t bytes;
  KarpoAttnArgs fwd;
};

int unpacked_of(const KarpoCacheAttendArgs* a, Unpacked* u) {
  // (with a window, each request's rows begin at a multiple of 32)
  int64_t rows = seen_keys(a);
  if (rows < a->total_keys) {
    rows += (int64_t)(kCacheGroup - 1) * a->n_seq;
    if (rows > a->total_keys) rows = a->total_keys;
  }
  if (rows < 1) rows = 1;  // (a key bound of 0 would not be checked)
  const int64_t row_bytes = 2 * (int64_t)a->cache.kv_heads * a->cache.head_dim;
  u->rows = rows;
  u->k_offset = round_up(4 * ((int64_t)a->n_seq + 1), 256);
  u->v_offset = u->k_offset + round_up(rows * row_bytes, 256);
  u->ws_offset = u->v_offset + round_up(rows * row_bytes, 256);
  KarpoAttnArgs& f = u->fwd;
  memset(&f, 0, sizeof(f));
  f.q = a->q;
  f.o = a->o;
  f.q_stride_tok = a->q_stride_tok;
  f.q_stride_head = a->q_stride_head;
  f.o_stride_tok = a->o_stride_tok;
  f.o_stride_head = a->o_stride_head;
  f.k_stride_tok = f.v_stride_tok = (int64_t)a->cache.kv_heads * a->cache.head_dim;
  f.k_stride_head = f.v_stride_head = a->cache.head_dim;
  f.q_cu = a->q_cu;
  f.n_seq = a->n_seq;
  f.heads = a->heads;
  f.kv_heads = a->cache.kv_heads;
  f.head_dim = a->cache.head_dim;
  f.total_q = a->total_q;
  f.max_q = a->max_q;
  f.scale = a->scale;
  f.window_left = a->window_left;
  f.window_right = a->window_right;
  f.key_bound = rows;
  size_t ws = 0;
  const int st = karpo_attn_workspace_bytes(&f, &ws);
  if (st != KARPO_ATTN_OK) return st;
  u->bytes = (size_t)u->ws_offset + ws;
  return KARPO_ATTN_OK;
}

// Sizes and head counts (everything the workspace's size depends on).
int check_attend(const KarpoCacheAttendArgs* a, CacheRef* c, CacheRows* r) {
  if (a == nullptr) return KARPO_ATTN_ERR_NULL;
  int st = check_cache(a->cache, c);
  if (st != KARPO_ATTN_OK) return st;
  st = check_rows(a->table, a->table_stride, a->width, a->lengths, a->n_seq, a->cache.block_size, r);
  if (st != KARPO_ATTN_OK) return st;
  if (a->heads < 1 || a->heads % a->cache.kv_heads != 0) return KARPO_ATTN_ERR_HEADS;
  if (a->window_left < -1 || a->window_right < -1) return KARPO_ATTN_ERR_WINDOW;
  if (a->total_q < 0 || a->max_q < 0 || a->total_keys < 0 || a->total_keys > INT32_MAX) return KARPO_ATTN_ERR_ARG;
  return KARPO_ATTN_OK;
}

// Whether the split path, which walks the keys once for each tile of query vectors, is the faster one; the other unpacks the
// keys and values first and has four launches. Both estimated in microseconds from the sizes, as measured: the split path's
// walks (a tile holds 64 vectors, 32 at head size 256, 16 at 512), and the unpacking at the memory's rate and the packed
// attention at the rate that it reaches with many query tiles, or with few of one or two requests. Of 198 shapes (head sizes
// 64 to 512, 1 to 16 requests of 700 to 32,768 tokens, 16 to 4,096 vectors) the rule's choice is over 15% slower than the
// other for two. Unpacked against split:
//   one request of 32,768 tokens, 16 key/value heads of 128: 128 vectors 166, 71 us; 512 vectors 307, 210; 1,024 458, 392
//   16 requests of 2,048: 128 vectors 102, 80; 256 vectors 117, 123; 512 vectors 165, 209
//   8 heads of 256: one request, 256 vectors 210, 134; 1,024 vectors 443, 474; 16 requests, 128 vectors 119, 88; 256 143, 149
//   4 heads of 512: one request, 512 vectors 284, 282; 1,024 vectors 436, 542; 16 requests, 512 vectors 251, 280
//   one request of 2,000 tokens: 16 heads of 128, 1,024 vectors 62, 52; 8 of 256, 71, 54; 4 of 512, 78, 56
bool split(const KarpoCacheAttendArgs* a) {
  const int d = a->cache.head_dim;
  const double vectors = (double)a->max_q * (a->heads / a->cache.kv_heads);
  if (vectors <= 64) return true;
  if (vectors >= 1 << 15) return false;  // (position_of holds below 2^16)
  const double keys = (double)seen_keys(a) * a->cache.kv_heads, tile = d <= 128 ? 64 : d == 256 ? 32 : 16;
  if (ceil(vectors / tile) * a->cache.kv_heads > 65535) return false;  // (a launch's second dimension)
  const double walk = d == 64 ? 3.5e-5 : d == 128 ? 4.6e-5 : d == 256 ? 5.3e-5 : 6.1e-5;
  const double query_tiles = a->n_seq * ceil(vectors / 128) * a->cache.kv_heads;
  const double most = d == 512 ? 0.8e9 : 1.3e9, few = 0.35e9 + 0.5e6 * vectors;  // operations a microsecond
  const double rate = a->n_seq <= 2 && query_tiles < 256 && few < most ? few : most;
  const double by_split = 17 + keys * (walk * ceil(vectors / tile) + (a->n_seq > 1 ? 3e-5 : 0));
  const double unpacked = 33 + keys * d * 0.9e-6 + 4 * vectors * keys * d / rate;
  return by_split <= unpacked;
}

AttendShape shape_of(const KarpoCacheAttendArgs* a, const CacheRef& c, const CacheRows& r) {
  int64_t seen = a->total_keys < r.most ? a->total_keys : r.most;
  if (a->window_left >= 0 && (int64_t)a->max_q + a->window_left < seen) seen = (int64_t)a->max_q + a->window_left;
  return attend_shape(c, a->n_seq, a->heads / a->cache.kv_heads, a->max_q, seen);
}

}  // namespace

extern "C" int karpo_cache_attend_workspace_bytes(const KarpoCacheAttendArgs* a, size_t* bytes) {
  CacheRef c;
  CacheRows r;
  const int st = check_attend(a, &c, &r);
  if (st != KARPO_ATTN_OK) return st;
  if (bytes == nullptr) return KARPO_ATTN_ERR_NULL;
  if (split(a)) {
    *bytes = (size_t)shape_of(a, c, r).bytes;
    return KARPO_ATTN_OK;
  }
  Unpacked u;
  const int su = unpacked_of(a, &u);
  if (su != KARPO_ATTN_OK) return su;
  *bytes = u.bytes;
  return KARPO_ATTN_OK;
}

extern "C" int karpo_cache_attend(const KarpoCacheAttendArgs* a, void* stream) {
  ReadParams p;
  memset(&p, 0, sizeof(p));
  int st = check_attend(a, &p.c, &p.r);
  if (st != KARPO_ATTN_OK) return st;
  if (a->total_q == 0 || a->n_seq == 0 || a->max_q == 0) return KARPO_ATTN_OK;
  if (!a->q || !a->o || !a->q_cu) return KARPO_ATTN_ERR_NULL;
  if (!row_strides(a->q, a->q_stride_tok, a->q_stride_head) || !row_strides(a->o, a->o_stride_tok, a->o_stride_head))
    return KARPO_ATTN_ERR_LAYOUT;
  if (split(a)) {
    const AttendShape shape = shape_of(a, p.c, p.r);
    if (shape.bytes > 0 &&
        (a->workspace == nullptr || a->workspace_bytes < (size_t)shape.bytes || !aligned(a->workspace, 16)))
      return KARPO_ATTN_ERR_WORKSPACE;
    AttendParams t;
    memset(&t, 0, sizeof(t));
    t.c = p.c;
    t.r = p.r;
    t.q = static_cast<const uint16_t*>(a->q);
    t.o = static_cast<uint16_t*>(a->o);
    t.sq_t = a->q_stride_tok;
    t.sq_h = a->q_stride_head;
    t.so_t = a->o_stride_tok;
    t.so_h = a->o_stride_head;
    t.q_cu = a->q_cu;
    t.total_q = a->total_q;
    t.max_q = a->max_q;
    t.group = a->heads / a->cache.kv_heads;
    t.left = a->window_left >= kMostTokens ? -1 : a->window_left;  // (sees everything, and stays within 32 bits)
    t.right = a->window_right;
    t.scale = fabsf(a->scale) * 1.4426950408889634f;
    if (t.scale < 1e-30f) t.scale = 1e-30f;  // (NaN stays)
    t.sign = a->scale < 0.f ? 0x80008000u : 0u;
    t.per_group = 1.f / t.group;
    t.whole = shape.whole;
    t.parts = shape.parts;
    if (!shape.whole) {
      t.units = static_cast<int32_t*>(a->workspace);
      t.partial = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + shape.units_bytes);
    }
    if (launch_cache_attend(t, shape, static_cast<hipStream_t>(stream)) != hipSuccess) return KARPO_ATTN_ERR_LAUNCH;
    return KARPO_ATTN_OK;
  }
  Unpacked u;
  st = unpacked_of(a, &u);
  if (st != KARPO_ATTN_OK) return st;
  if (a->workspace == nullptr || a->workspace_bytes < u.bytes || !aligned(a->workspace, 16))
    return KARPO_ATTN_ERR_WORKSPACE;
  char* const ws = static_cast<char*>(a->workspace);
  p.q_cu = a->q_cu;
  p.window_left = a->window_left;
  p.max_q = a->max_q;
  p.total_q = a->total_q;
  p.o = static_cast<uint16_t*>(a->o);
  p.so_t = a->o_stride_tok;
  p.so_h = a->o_stride_head;
  p.heads = a->heads;
  p.no_scale = isnan(a->scale);  // (the packed attention takes a NaN for the least scale)
  p.k = reinterpret_cast<uint16_t*>(ws + u.k_offset);
  p.v = reinterpret_cast<uint16_t*>(ws + u.v_offset);
  p.rows = u.rows;
  p.k_cu = reinterpret_cast<int32_t*>(ws);
  if (launch_cache_read(p, static_cast<hipStream_t>(stream)) != hipSuccess) return KARPO_ATTN_ERR_LAUNCH;
  if (p.no_scale) return KARPO_ATTN_OK;
  u.fwd.k = p.k;
  u.fwd.v = p.v;
  u.fwd.k_cu = p.k_cu;
  u.fwd.workspace = ws + u.ws_offset;
  u.fwd.workspace_bytes = a->workspace_bytes - (size_t)u.ws_offset;
  return karpo_attn_fwd(&u.fwd, stream);
}
