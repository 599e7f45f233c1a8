/*
 * C ABI of libfa_paged_attention.so for latent attention: a token's keys and values of all heads come from
 * one shared latent vector c (latent_dim elements) and one rotated key part r (rope_dim elements), and
 * the paged pool holds the row [c, r] of each token, once for all heads.
 *
 *   fa_latent_cache_append        normalises the latents, rotates key parts and queries, stores the rows
 *   fa_latent_cache_gather        rows of the pool, read back as dense 16-bit rows
 *   fa_paged_attention_latent     attention over the pool itself: the products that expand keys and values
 *                                 are absorbed into the queries before it and the results after it
 *   fa_attention_latent_expanded  causal attention over keys and values that have been expanded for each
 *                                 head, the rotated key part shared by the heads
 *
 * A batch is described as in fa_ragged.h: query_start [num_seqs + 1], context_lens [num_seqs] with the
 * new tokens, block_tables [num_seqs, max_blocks_per_seq], all int32 in device memory; token j of a sequence's n sits
 * at position context_lens[s] - n + j and sees the keys 0 .. that position.  Block ids outside the pool are never
 * read from or written to (reads take a block of the pool instead, writes are left out); a token at a negative position
 * sees nothing, and its result is zero; one at a position past the table's columns is not stored, and attends as one
 * at the table's last position would.
 *
 * Pools: row t of block b begins at base + b * block_stride + t * token_stride (elements) and holds latent_dim +
 * rope_dim contiguous ones: 16-bit of the queries' type, or E4M3 bytes, each standing for itself times its row's
 * scale, scales[b * block_size + t].  Rows of the pool that no token sees, and their scales, may hold
 * anything.  A row of a new token that holds infinities or NaN can reach earlier new tokens of its sequence
 * in the same call.  Scales are positive; next to a row whose scale is 2^100 attention counts weights
 * down to 2^-32 of the largest, next to one of 2^120 down to 2^-12.  latent_dim is 256 or 512, rope_dim 64.
 *
 * Nothing but kernel launches is put on options->stream unless options->elapsed_us is given.  Of options these entries read
 * stream, elapsed_us (1 float) and validate_only.  No exception crosses this boundary.
 */
#ifndef FA_LATENT_H_
#define FA_LATENT_H_

#include <stdint.h>

#include "fa_kv_cache.h"
#include "fa_paged_attention.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct fa_latent_append_shape {
  uint32_t struct_size;        /* sizeof(fa_latent_append_shape) in the caller's header */
  int32_t num_seqs;
  int32_t num_tokens;
  int32_t num_heads;           /* query heads; not looked at without query_rope */
  int32_t latent_dim;
  int32_t rope_dim;
  int32_t block_size;          /* power of two >= 16 */
  int32_t max_blocks_per_seq;
  int64_t block_stride, token_stride;          /* of the pool, in elements */
  int64_t latent_token_stride, rope_key_token_stride;
  int64_t query_token_stride, query_head_stride;
  int64_t query_out_token_stride, query_out_head_stride;
  int32_t src_dtype;           /* fa_dtype of latent, rope_key, query_rope and query_rope_out */
  int32_t cache_dtype;         /* FA_KV_CACHE_16BIT or FA_KV_CACHE_E4M3 */
  int32_t num_pool_blocks;
  int32_t max_positions;       /* rows of cos_sin; 0: nothing is rotated */
  int32_t interleaved;         /* pairs: 0 elements k and rope_dim / 2 + k, 1 elements 2k and 2k + 1 */
  float norm_eps;
} fa_latent_append_shape;
#define FA_LATENT_APPEND_SHAPE_INIT {(uint32_t)sizeof(fa_latent_append_shape)}

/*
 * latent      [num_tokens, latent_dim]; with norm_weight [latent_dim] (fp32) a row c becomes
 *             c / sqrt(mean(c^2) + norm_eps) * norm_weight, in 32 bits; without, it stays as it is
 * rope_key    [num_tokens, rope_dim], and query_rope [num_tokens, num_heads, rope_dim] -> query_rope_out (which may be
 *             query_rope itself; both NULL: the rows only): rotated by the row of cos_sin [max_positions, rope_dim] (fp32:
 *             the cosines of a position's angles, then their sines), in 32 bits; a position beyond the table takes its last row
 * scales      [num_pool_blocks, block_size], written for E4M3 pools: the least power of two from 2^-100 on that brings the row's
 *             largest magnitude (latent and key part together) to 448 or less; bytes are rounded to nearest even
 * Rows are rounded once, when they are stored.  A new token's place must be its own: two tokens for one row race.
 */
int32_t fa_latent_cache_append(const void *latent, const void *rope_key, void *cache, const float *norm_weight, const float *cos_sin,
                               const void *query_rope, void *query_rope_out, float *scales, const int32_t *block_tables,
                               const int32_t *query_start, const int32_t *context_lens, const fa_latent_append_shape *shape,
                               const fa_paged_attention_options *options);

typedef struct fa_latent_gather_shape {
  uint32_t struct_size;        /* sizeof(fa_latent_gather_shape) in the caller's header */
  int32_t num_seqs;
  int32_t num_rows;
  int32_t latent_dim;
  int32_t rope_dim;
  int32_t block_size;
  int32_t max_blocks_per_seq;
  int32_t num_pool_blocks;
  int64_t block_stride, token_stride;
  int64_t out_stride;          /* elements from row to row of out */
  int32_t out_dtype;           /* fa_dtype of out, and of a 16-bit pool */
  int32_t cache_dtype;
} fa_latent_gather_shape;
#define FA_LATENT_GATHER_SHAPE_INIT {(uint32_t)sizeof(fa_latent_gather_shape)}

/*
 * out [num_rows, latent_dim + rope_dim]: row row_start[s] + i becomes key first_keys[s] + i of sequence s, for every i below
 * row_start[s + 1] - row_start[s] (row_start [num_seqs + 1], ascending; first_keys [num_seqs], NULL: 0).  A key
 * before 0, past the table's columns or in a block outside the pool gives zeros; rows of out beyond the last sequence's stay as
 * they are.
 */
int32_t fa_latent_cache_gather(void *out, const void *cache, const float *scales, const int32_t *block_tables, const int32_t *row_start,
                               const int32_t *first_keys, const fa_latent_gather_shape *shape, const fa_paged_attention_options *options);

typedef struct fa_latent_attention_shape {
  uint32_t struct_size;        /* sizeof(fa_latent_attention_shape) in the caller's header */
  int32_t num_seqs;
  int32_t num_tokens;
  int32_t num_heads;
  int32_t latent_dim;
  int32_t rope_dim;
  int32_t block_size;
  int32_t max_blocks_per_seq;
  int64_t block_stride, token_stride;          /* of the pool, in elements, of 16-byte multiples */
  int64_t query_latent_token_stride, query_latent_head_stride;
  int64_t query_rope_token_stride, query_rope_head_stride;
  int64_t out_token_stride, out_head_stride;
  int32_t q_dtype;             /* fa_dtype of queries and out */
  int32_t cache_dtype;         /* FA_KV_CACHE_16BIT or FA_KV_CACHE_E4M3 */
  int32_t num_pool_blocks;
  int32_t max_query_len;       /* no sequence brings more new tokens; > 0 */
  int32_t max_context_len;     /* no sequence has more keys; 0: what the block table holds */
} fa_latent_attention_shape;
#define FA_LATENT_ATTENTION_SHAPE_INIT {(uint32_t)sizeof(fa_latent_attention_shape)}

/* Device memory that a call of this shape works in (16-byte aligned, any contents).  0 for a shape that a call would refuse. */
int64_t fa_paged_attention_latent_workspace_bytes(const fa_latent_attention_shape *shape);

/*
 * With c, r the parts of a cached row:
 *   s   = scale (query_latent . c + query_rope . r)
 *   out = sum of softmax(s) c                           [num_tokens, num_heads, latent_dim]
 * Tokens beyond max_query_len of their sequence are left out, their rows of out stay as they are; so do rows behind the last sequence's.
 */
int32_t fa_paged_attention_latent(void *out, const void *query_latent, const void *query_rope, const void *cache, const float *scales,
                                  const int32_t *block_tables, const int32_t *query_start, const int32_t *context_lens, float scale,
                                  void *workspace, int64_t workspace_bytes, const fa_latent_attention_shape *shape,
                                  const fa_paged_attention_options *options);

typedef struct fa_latent_expanded_shape {
  uint32_t struct_size;        /* sizeof(fa_latent_expanded_shape) in the caller's header */
  int32_t num_seqs;
  int32_t num_tokens;
  int32_t num_keys;
  int32_t num_heads;
  int32_t head_size;           /* of expanded keys and values: 64 or 128 */
  int32_t rope_dim;            /* 64 */
  int32_t dtype;               /* fa_dtype of everything */
  int64_t query_token_stride, query_head_stride;
  int64_t key_token_stride, key_head_stride;
  int64_t rope_key_token_stride;
  int64_t value_token_stride, value_head_stride;
  int64_t out_token_stride, out_head_stride;
  int32_t max_query_len;       /* no sequence brings more new tokens; > 0 */
  int32_t max_key_len;         /* no sequence has more keys; 0: num_keys */
} fa_latent_expanded_shape;
#define FA_LATENT_EXPANDED_SHAPE_INIT {(uint32_t)sizeof(fa_latent_expanded_shape)}

/* Device memory that a call of this shape works in (16-byte aligned, any contents).  0 for a shape that a call would refuse. */
int64_t fa_attention_latent_expanded_workspace_bytes(const fa_latent_expanded_shape *shape);

/*
 * query [num_tokens, num_heads, head_size + rope_dim], key and value [num_keys, num_heads, head_size], rope_key [num_keys,
 * rope_dim], out [num_tokens, num_heads, head_size].  Sequence s has the tokens query_start[s] .. and the keys key_start[s] ..
 * (both [num_seqs + 1], ascending); its last token is at its last key, and a token sees the keys up to its own.
 *   s   = scale (query[:head_size] . key + query[head_size:] . rope_key)
 *   out = sum of softmax(s) value
 * A token that sees no key gets zeros.  Tokens beyond max_query_len of their sequence are left out, their rows of out stay as they are;
 * of keys beyond max_key_len nothing is read.  Values of a new token that are infinite or NaN can reach earlier new tokens
 * of its sequence (their weight is zero, and the product is not); nothing reaches another sequence.
 */
int32_t fa_attention_latent_expanded(void *out, const void *query, const void *key, const void *rope_key, const void *value,
                                     const int32_t *query_start, const int32_t *key_start, float scale, void *workspace,
                                     int64_t workspace_bytes, const fa_latent_expanded_shape *shape,
                                     const fa_paged_attention_options *options);

#ifdef __cplusplus
}
#endif

#endif /* FA_LATENT_H_ */
