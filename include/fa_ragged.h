/*
 * C ABI of libfa_paged_attention.so for ragged batches: each call brings the new tokens of all its
 * sequences, any number of each (one token of a running sequence, a whole prompt, a piece of
 * one), one behind the other in arrays of num_tokens rows.
 *
 *   fa_kv_cache_append               rotates queries and keys by their positions and puts keys and
 *                                    values into the paged pools; pools of integers keep a scale
 *                                    for each block and kv head up to date
 *   fa_paged_attention_ragged        causal attention of the new tokens over the pools
 *   fa_paged_attention_differential  the difference of two softmax maps over one cache, each
 *                                    head's result normalised
 *
 * Arrays that describe the batch (device memory):
 *   query_start   [num_seqs + 1] int32, ascending: tokens query_start[s] .. query_start[s+1] - 1
 *                 are sequence s's (none, if the two are equal)
 *   context_lens  [num_seqs] int32: keys of the sequence WITH its new tokens; token j of n sits
 *                 at position context_lens[s] - n + j and sees the keys 0 .. that position
 *   block_tables  [num_seqs, max_blocks_per_seq] int32
 * Block ids outside the pool are never read from or written to (reads take a block of the pool
 * instead, writes are left out); a token at a negative position (context_lens[s] < n) is not stored
 * and its result is zero; one at a position past the table's columns is not stored either, and
 * attends as one at the table's last position would.
 * Pool rows that none of the call's tokens sees -- past the context, before every token's window,
 * unused blocks -- and scales of such blocks may hold anything.  Keys that a token does not see
 * have no weight whatever they are; values of one new token that are infinite or NaN can reach earlier
 * new tokens of its sequence in the same call, whose weight for them is zero, as products of zero.
 *
 * Pools are addressed as in fa_paged_attention.h.  Nothing but kernel launches is put on
 * options->stream unless options->elapsed_us is given.  No exception crosses this boundary.
 */
#ifndef FA_RAGGED_H_
#define FA_RAGGED_H_

#include <stdint.h>

#include "fa_kv_cache.h"
#include "fa_paged_attention.h"

#ifdef __cplusplus
extern "C" {
#endif

/* A further fa_kv_cache_dtype, of the entries in this header only: integers -127 .. 127, each
 * standing for itself times the scale of its block and kv head. */
#define FA_KV_CACHE_I8 3

typedef struct fa_kv_cache_append_shape {
  uint32_t struct_size;        /* sizeof(fa_kv_cache_append_shape) in the caller's header */
  int32_t num_seqs;
  int32_t num_tokens;
  int32_t num_heads;           /* query heads; not looked at without query */
  int32_t num_kv_heads;
  int32_t head_size;           /* multiple of 16, at most 1024 */
  int32_t block_size;          /* power of two >= 16 */
  int32_t max_blocks_per_seq;
  int64_t kv_block_stride;     /* strides in elements; rows of head_size elements are contiguous */
  int64_t kv_token_stride;
  int64_t kv_head_stride;
  int64_t query_token_stride, query_head_stride;
  int64_t query_out_token_stride, query_out_head_stride;
  int64_t key_token_stride, key_head_stride;
  int64_t value_token_stride, value_head_stride;
  int32_t src_dtype;           /* fa_dtype of query, query_out, key and value */
  int32_t cache_dtype;         /* fa_kv_cache_dtype, or FA_KV_CACHE_I8 */
  int32_t kv_scale_mode;       /* FP8 pools: FA_KV_SCALE_TENSOR or FA_KV_SCALE_HEAD; integers: FA_KV_SCALE_BLOCK */
  int32_t num_pool_blocks;
  int32_t max_positions;       /* rows of cos_sin */
  int32_t rotary_dim;          /* rotated elements of a row, the first ones: multiple of 16; 0: none */
  int32_t interleaved;         /* pairs: 0 elements k and rotary_dim / 2 + k, 1 elements 2k and 2k + 1 */
  float fp8_scale;             /* of FA_KV_SCALE_TENSOR; 0 means 1 */
} fa_kv_cache_append_shape;
#define FA_KV_CACHE_APPEND_SHAPE_INIT {(uint32_t)sizeof(fa_kv_cache_append_shape)}

/*
 * cos_sin   [max_positions, rotary_dim] fp32: the cosines of a position's rotary_dim / 2 angles,
 *           then their sines; NULL with rotary_dim 0.  A pair (a, b) becomes
 *           (a cos - b sin, b cos + a sin), in 32 bits, each operation rounded by itself; the
 *           result is rounded to the query type, or to a byte, once.  A position beyond the
 *           table takes its last row.
 * query     [num_tokens, num_heads, head_size], rotated into query_out, which may be query itself;
 *           both NULL: keys and values only.
 * k_scales, v_scales   FA_KV_SCALE_HEAD: [num_kv_heads], read.  FA_KV_SCALE_BLOCK:
 *           [num_pool_blocks, num_kv_heads], read and written: the scale of a block that gets new
 *           rows becomes max(scale, max|x| * (1 / 127) over them, 2^-126), where a block whose first
 *           row is new starts from 0; rows that were there are rounded again, to
 *           rint(byte * (old scale / new scale)), and new ones are rint(x * (1 / scale)).
 * Each new token's place must belong to its sequence alone: two tokens for one row, or new rows of
 * two sequences in one block of integers, race.
 * Of options this entry reads stream, elapsed_us (1 float) and validate_only.
 */
int32_t fa_kv_cache_append(const void *query, void *query_out, const void *key, const void *value, void *key_cache,
                           void *value_cache, const float *cos_sin, const int32_t *block_tables,
                           const int32_t *query_start, const int32_t *context_lens, float *k_scales, float *v_scales,
                           const fa_kv_cache_append_shape *shape, const fa_paged_attention_options *options);

typedef struct fa_ragged_shape {
  uint32_t struct_size;        /* sizeof(fa_ragged_shape) in the caller's header */
  int32_t num_seqs;
  int32_t num_tokens;
  int32_t num_heads;           /* at most 16 per kv head */
  int32_t num_kv_heads;
  int32_t head_size;           /* elements of a cache row: 64 or 128 (differential: two query / key halves of 32 or 64) */
  int32_t block_size;          /* power of two >= 16 */
  int32_t max_blocks_per_seq;
  int64_t kv_block_stride;     /* strides in elements, of 16-byte multiples */
  int64_t kv_token_stride;
  int64_t kv_head_stride;
  int64_t query_token_stride, query_head_stride;
  int32_t q_dtype;             /* fa_dtype of query and out */
  int32_t cache_dtype;         /* FA_KV_CACHE_16BIT (q_dtype elements), _E5M2, _E4M3 or FA_KV_CACHE_I8 */
  int32_t num_pool_blocks;     /* > 0 */
  int32_t max_query_len;       /* no sequence brings more new tokens; > 0 */
  int32_t max_context_len;     /* no sequence has more keys; 0: what the block table holds */
} fa_ragged_shape;
#define FA_RAGGED_SHAPE_INIT {(uint32_t)sizeof(fa_ragged_shape)}

/* Device memory that a call of this shape works in (16-byte aligned, any contents); maps: 1 for
 * fa_paged_attention_ragged, 2 for fa_paged_attention_differential.  0 for a shape that a call would refuse. */
int64_t fa_paged_attention_ragged_workspace_bytes(const fa_ragged_shape *shape, int32_t maps);

/*
 * out [num_tokens, num_heads, head_size], contiguous, q_dtype.  Of options: sinks, alibi_slopes,
 * softcap, mask_flags and window_left as in fa_paged_attention.h; fp8_scale, kv_scale_mode,
 * k_scales and v_scales of byte pools (integers take FA_KV_SCALE_BLOCK or _HEAD; scales are not negative, and 0
 * stands for rows of zeros); stream, elapsed_us (1 float) and validate_only.  A token that sees no key gets zeros.  Tokens beyond max_query_len of their
 * sequence are left out.
 */
int32_t fa_paged_attention_ragged(void *out, const void *query, const void *key_cache, const void *value_cache,
                                  const int32_t *block_tables, const int32_t *query_start, const int32_t *context_lens,
                                  float scale, void *workspace, int64_t workspace_bytes, const fa_ragged_shape *shape,
                                  const fa_paged_attention_options *options);

/*
 * With q1, q2 the halves of a query row and k1, k2 those of a key row:
 *   o   = softmax(scale q1 k1^T) V - lambdas[head] softmax(scale q2 k2^T) V      (in 32 bits)
 *   out = out_scale * norm_weight * o / sqrt(mean(o^2) + norm_eps)
 * lambdas [num_heads], norm_weight [head_size] fp32 device memory; without norm_weight
 * out = out_scale * o.  Rows of zeros stay zeros, also with norm_eps 0.  16-bit and integer pools; of mask_flags only FA_MASK_WINDOW; no sinks.
 */
int32_t fa_paged_attention_differential(void *out, const void *query, const void *key_cache, const void *value_cache,
                                        const int32_t *block_tables, const int32_t *query_start,
                                        const int32_t *context_lens, float scale, const float *lambdas,
                                        const float *norm_weight, float norm_eps, float out_scale, void *workspace,
                                        int64_t workspace_bytes, const fa_ragged_shape *shape,
                                        const fa_paged_attention_options *options);

#ifdef __cplusplus
}
#endif

#endif /* FA_RAGGED_H_ */
