/*
 * karpo_cache4.h - C ABI of the MI355X (gfx950) block cache in 4 bits: the operators of karpo_cache.h over keys and values of
 * half the size. karpo_cache_reserve serves both (its tables, slots and writes know no format).
 *
 *   karpo_cache4_append  new keys and values into their blocks, normed and rotated on the way where asked
 *   karpo_cache4_read    cached rows of a batch back as packed bf16 keys and values
 *   karpo_cache4_attend  packed attention of new queries over cached keys
 *
 * An element is an e2m1 code (0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives) times a power of two 2^e that 32 consecutive
 * elements of one token's head share, kept as a byte e + 127: 4.25 bits an element, and a bf16 value exactly. e is the least
 * exponent with max|finite element| <= 6 * 2^e, within KARPO_CACHE4_MIN_EXP .. MAX_EXP; codes are the nearest, ties to even, an
 * element past the range is stored at its end, an infinity too; a NaN makes its 32 elements NaN (the byte is 255). A token's
 * scales are its own: appending leaves the block's other tokens as they are.
 * The pool need not be initialised: what a slot holds that no append wrote (bytes of 253 and 254 too, which append never writes)
 * reaches no query that does not see its token.
 *
 * Layout (token t and element d within a block of one head; h = t / 32, an even element in the lower half of its byte):
 *   keys    h * 16 D + ((t / 16 % 2) * (D / 32) + d / 32) * 256 + (t % 16) * 16 + d % 32 / 2
 *   values  h * 16 D + ((d / 64) * 64 + (t / 4 % 4) * 16 + d / 2 % 16) * 16 + (d / 32 % 2) * 8 + (t / 16 % 2) * 4 + t % 4
 *   scales  h * 2 D + (keys) ((d / 32 % 4) * 16 + t % 16) * (D / 64) + (d / 128) * 2 + t / 16 % 2, at head size 64
 *           ((t / 16 % 2) * 2 + d / 32) * 16 + t % 16; (values) D + (d / 32) * 32 + (t / 4 % 4) * 8 + (t / 16 % 2) * 4 + t % 4
 * so that 16 bytes of keys are one lane's operand of a 16x16x128 scaled matrix instruction and 16 bytes of values four of a
 * 16x16x32 one.
 *
 * In attention the keys' codes enter the matrix instruction as they are, the queries (bf16) as two e4m3 terms under powers of two
 * of their own (2^-22 of the largest of 32 elements off); softmax statistics, sums and weights are those of karpo_cache_attend.
 * Everything else, and what happens where bounds, tables or lengths do not hold, is as in karpo_cache.h.
 */
#ifndef KARPO_CACHE4_H
#define KARPO_CACHE4_H

#include <stddef.h>
#include <stdint.h>

#include "karpo_cache.h"

#ifdef __cplusplus
extern "C" {
#endif

#define KARPO_CACHE4_MIN_EXP (-100)
#define KARPO_CACHE4_MAX_EXP 125

typedef struct KarpoCache4 {
  void* keys;   /* device, apart from values, [blocks][kv_heads][block_size * head_dim / 2] bytes, 16-byte aligned */
  void* values; /* the same */
  void* scales; /* device, [blocks][kv_heads][block_size / 32][2][head_dim] bytes, 16-byte aligned */
  int64_t blocks;
  int32_t kv_heads;
  int32_t head_dim;   /* 64, 128, 256 or 512 */
  int32_t block_size; /* 32, 64 or 128 tokens */
} KarpoCache4;

/* The fields are those of the structures of karpo_cache.h. */
typedef struct KarpoCache4AppendArgs {
  KarpoCache4 cache;
  const void* k;
  const void* v;
  int64_t k_stride_tok, k_stride_head, v_stride_tok, v_stride_head;
  int64_t rows;
  const int32_t* writes;
  int64_t n_writes;
  KarpoCachePrologue prologue; /* all zeros: rows as they are */
} KarpoCache4AppendArgs;

typedef struct KarpoCache4ReadArgs {
  KarpoCache4 cache;
  const int32_t* table;
  int64_t table_stride;
  int32_t width;
  int32_t n_seq;
  const int32_t* lengths;
  void* k;
  void* v;
  int64_t rows;
  int32_t* k_cu;
} KarpoCache4ReadArgs;

typedef struct KarpoCache4AttendArgs {
  KarpoCache4 cache;
  const void* q;
  void* o;
  int64_t q_stride_tok, q_stride_head, o_stride_tok, o_stride_head;
  const int32_t* q_cu;
  const int32_t* lengths;
  const int32_t* table;
  int64_t table_stride;
  int32_t width;
  int32_t n_seq;
  int32_t heads;
  int32_t max_q;
  int64_t total_q;
  int64_t total_keys;
  float scale;
  int32_t window_left, window_right;
  void* workspace;
  size_t workspace_bytes;
} KarpoCache4AttendArgs;

int karpo_cache4_append(const KarpoCache4AppendArgs* args, void* stream);
int karpo_cache4_read(const KarpoCache4ReadArgs* args, void* stream);

/* Bytes of workspace karpo_cache4_attend needs for these sizes (16-byte aligned; calls that overlap need their own). */
int karpo_cache4_attend_workspace_bytes(const KarpoCache4AttendArgs* args, size_t* bytes);
int karpo_cache4_attend(const KarpoCache4AttendArgs* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* KARPO_CACHE4_H */
