/*
 * karpo_cache.h - C ABI of the MI355X (gfx950) block cache: keys and values kept between calls in 8 bits, and the four
 * operators of a serving step over them.
 *
 *   karpo_cache_reserve  request lengths -> block table, slot map, positions and the list of block writes
 *   karpo_cache_append   new keys and values into their blocks
 *   karpo_cache_read     cached rows of a batch back as packed bf16 keys and values
 *   karpo_cache_attend   packed attention of new queries over cached keys
 *
 * A cache is a pool of blocks of `block_size` tokens. A block holds, for each key/value head, its tokens' keys and values
 * as e4m3 codes and one scale 2^e for the keys and one for the values: an element is code * 2^e, which bf16 holds exactly.
 * e is the least exponent with max|finite element written| <= 448 * 2^e, within KARPO_CACHE_MIN_EXP .. MAX_EXP (an
 * element past the range is stored at its end, an infinity too; NaN stays NaN). A power of two costs an e4m3 element no
 * precision against a free scale, and makes scaling exact, also where a block's scale grows: its earlier codes are then
 * rounded again, code' = e4m3(code * 2^(e_old - e_new)).
 *
 * Layout (bytes; token t and element d within the block, one head's keys or values are block_size * head_dim bytes):
 *   keys    ((t / 16) * (D / 64) + d / 64) * 1024 + (t % 16) * 64 + d % 64
 *   values  (t / 32) * 32 D + (d / 32) * 1024 + (d % 16) * 64 + (t / 4 % 4) * 16 + (d / 16 % 2) * 8 + (t / 16 % 2) * 4 + t % 4
 * so that 16 consecutive bytes are one lane's operand of two 16x16x32 matrix instructions.
 *
 * A request's cached tokens 0 .. length - 1 lie in the blocks table[0], table[1], ...; token p in slot p % block_size of
 * table[p / block_size]. Block ids outside the pool are never followed: such tokens read as zeros and are not written.
 * Lengths below 0 count as 0, lengths past the table's row as the row's tokens.
 *
 * Softmax statistics and sums are fp32. The weights enter the second product as two bf16 terms (2^-17 off) for few queries, and
 * as one (2^-8) in long chunks, whose keys are unpacked for karpo_attn_fwd; which of the two goes by the sizes.
 *
 * Conventions are those of karpo_attn.h: device pointers, sizes and strides in elements, launches on the given stream
 * only, no allocation, no synchronisation, failures as KARPO_ATTN_* status codes (karpo_attn_strerror). Lengths, bounds,
 * tables and writes are read when the kernels run, so that a captured graph sees what they hold at each replay.
 */
#ifndef KARPO_CACHE_H
#define KARPO_CACHE_H

#include <stddef.h>
#include <stdint.h>

#include "karpo_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

#define KARPO_CACHE_MIN_EXP (-100)
#define KARPO_CACHE_MAX_EXP 119

/* karpo_cache_reserve's status word (device). */
#define KARPO_CACHE_NO_BLOCKS 10 /* the free list holds fewer blocks than the new tokens need */
#define KARPO_CACHE_BAD_LENGTHS 11 /* negative lengths or counts, counts past `rows`, tokens past the table's row, or a
                                      free_count outside the list */

typedef struct KarpoCache {
  void* keys;        /* device, apart from values, [blocks][kv_heads][block_size * head_dim] e4m3, 16-byte aligned */
  void* values;      /* the same */
  float* scales;     /* device, [blocks][kv_heads][2] fp32: 2^e of the keys, of the values; 8-byte aligned */
  int64_t blocks;
  int32_t kv_heads;
  int32_t head_dim;   /* 64, 128, 256 or 512 */
  int32_t block_size; /* 32, 64 or 128 tokens */
} KarpoCache;

typedef struct KarpoCacheReserveArgs {
  int32_t* table; /* device, [n_seq] rows of `width` block ids; the entries of newly taken blocks are written */
  int64_t table_stride;
  int32_t width;
  int32_t n_seq;
  const int32_t* lengths; /* device, [n_seq]: tokens each request holds */
  const int32_t* counts;  /* device, [n_seq]: tokens each request gets */
  const int32_t* free_blocks; /* device, [free_capacity]: ids of free blocks, taken from the end of the first free_count */
  const int32_t* free_count;  /* device, [1] */
  int32_t free_capacity;
  int32_t block_size;
  int64_t rows; /* rows of slots and positions: a bound of the counts' sum */
  /* outputs, device; none of them may overlap an input */
  int32_t* q_cu;        /* [n_seq + 1]: the requests' bounds in the packed new tokens */
  int32_t* new_lengths; /* [n_seq]: lengths + counts */
  int64_t* slots;       /* [rows]: block id * block_size + slot of each new token, -1 behind the last */
  int32_t* positions;   /* [rows]: each new token's position in its request, 0 behind the last */
  int32_t* writes;      /* [writes_capacity][4]: (block id, first slot, first row, tokens), 16-byte aligned; tokens 0: none */
  int64_t writes_capacity; /* karpo_cache_writes_capacity's */
  int32_t* free_left;   /* [1]: free_count less the blocks taken */
  int32_t* status;      /* [1]: 0, or why nothing was reserved (table untouched, q_cu 0, slots -1, no writes) */
} KarpoCacheReserveArgs;

typedef struct KarpoCacheAppendArgs {
  KarpoCache cache;
  const void* k; /* device, [rows][kv_heads][head_dim] bf16, head_dim contiguous, strides multiples of 8 elements */
  const void* v;
  int64_t k_stride_tok, k_stride_head, v_stride_tok, v_stride_head;
  int64_t rows;
  const int32_t* writes; /* device, [n_writes][4] as karpo_cache_reserve lists them; no block twice */
  int64_t n_writes;
} KarpoCacheAppendArgs;

typedef struct KarpoCacheReadArgs {
  KarpoCache cache;
  const int32_t* table; /* device, [n_seq] rows of `width` block ids */
  int64_t table_stride;
  int32_t width;
  int32_t n_seq;
  const int32_t* lengths; /* device, [n_seq] */
  void* k;                /* device, [rows][kv_heads][head_dim] bf16, contiguous, 16-byte aligned */
  void* v;
  int64_t rows;  /* a bound of the lengths' sum; what lies past it is not written */
  int32_t* k_cu; /* device, [n_seq + 1]: the requests' bounds in k and v */
} KarpoCacheReadArgs;

typedef struct KarpoCacheAttendArgs {
  KarpoCache cache;
  const void* q; /* device, [total_q][heads][head_dim] bf16, head_dim contiguous, strides multiples of 8, 16-byte aligned */
  void* o;       /* the same; must not overlap q */
  int64_t q_stride_tok, q_stride_head, o_stride_tok, o_stride_head;
  const int32_t* q_cu;    /* device, [n_seq + 1]: query rows of each request */
  const int32_t* lengths; /* device, [n_seq]: cached tokens of each request, its queries' own tokens among them: query
                             row i of Lq sits at token i + length - Lq */
  const int32_t* table;
  int64_t table_stride;
  int32_t width;
  int32_t n_seq;
  int32_t heads; /* a multiple of cache.kv_heads */
  int32_t max_q; /* a bound of every request's query rows */
  int64_t total_q;
  int64_t total_keys; /* a bound of the lengths' sum: the keys of long query runs are unpacked into the workspace */
                      /* Where a bound does not hold, the rows that are not computed become NaN: a request's rows past its
                         first max_q or, where the keys are unpacked, the rows of all requests (for more tokens than
                         total_keys too). A request whose q_cu are not within 0 .. total_q in order has no rows; with
                         max_q 0 nothing is written at all. */
  float scale; /* NaN makes the rows of every request with tokens NaN */
  int32_t window_left, window_right; /* -1: unbounded; causal is window_right 0 */
  void* workspace;
  size_t workspace_bytes;
} KarpoCacheAttendArgs;

/* Entries that karpo_cache_reserve's list of writes can take for these sizes; 0 for sizes it does not take. */
int64_t karpo_cache_writes_capacity(int64_t rows, int32_t n_seq, int32_t block_size);

int karpo_cache_reserve(const KarpoCacheReserveArgs* args, void* stream);
int karpo_cache_append(const KarpoCacheAppendArgs* args, void* stream);
int karpo_cache_read(const KarpoCacheReadArgs* args, void* stream);

/* Bytes of workspace karpo_cache_attend needs for these sizes (16-byte aligned; calls that overlap need their own). */
int karpo_cache_attend_workspace_bytes(const KarpoCacheAttendArgs* args, size_t* bytes);
int karpo_cache_attend(const KarpoCacheAttendArgs* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* KARPO_CACHE_H */
