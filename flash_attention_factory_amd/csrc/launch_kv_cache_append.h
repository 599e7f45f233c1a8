// Host launcher of the ragged append (declared in include/fa_ragged.h): argument checks, work-group shapes.
#pragma once

#include <algorithm>

#include "../../include/fa_ragged.h"
#include "kv_cache_append_kernel.h"
#include "launch_common.h"

namespace fa {

inline fa_status launch_kv_cache_append(const void *query, void *query_out, const void *key, const void *value, void *key_cache,
                                        void *value_cache, const float *cos_sin, const int32_t *block_tables,
                                        const int32_t *query_start, const int32_t *context_lens, float *k_scales,
                                        float *v_scales, const fa_kv_cache_append_shape *s, const fa_paged_attention_options *o) {
  if (s->num_seqs < 0 || s->num_tokens < 0 || s->num_kv_heads <= 0 || s->num_pool_blocks <= 0 || s->max_blocks_per_seq <= 0)
    return fail(FA_ERR_BAD_SHAPE, "num_seqs and num_tokens must be >= 0; num_kv_heads, num_pool_blocks and max_blocks_per_seq positive");
  const bool nothing = s->num_tokens == 0 || s->num_seqs == 0;
  if (!nothing && (!key || !value || !key_cache || !value_cache || !block_tables || !query_start || !context_lens))
    return fail(FA_ERR_NULL_POINTER, "key, value, key_cache, value_cache, block_tables, query_start and context_lens must all be non-NULL");
  if (!nothing && (query == nullptr) != (query_out == nullptr))
    return fail(FA_ERR_NULL_POINTER, "query and query_out come together");
  if (s->src_dtype != FA_DTYPE_F16 && s->src_dtype != FA_DTYPE_BF16)
    return fail(FA_ERR_UNSUPPORTED_DTYPE, "src_dtype %d is neither fp16 (0) nor bf16 (1)", s->src_dtype);
  const int c = s->cache_dtype;
  if (c != FA_KV_CACHE_16BIT && c != FA_KV_CACHE_E5M2 && c != FA_KV_CACHE_E4M3 && c != FA_KV_CACHE_I8)
    return fail(FA_ERR_UNSUPPORTED_DTYPE, "cache_dtype %d is none of 16-bit (0), E5M2 (1), E4M3 (2), integers (3)", c);
  if (s->head_size <= 0 || s->head_size % 16 || s->head_size > 1024)
    return fail(FA_ERR_UNSUPPORTED_HEAD_OR_BLOCK_SIZE, "head_size %d must be a multiple of 16, at most 1024", s->head_size);
  if (s->block_size < 16 || !is_pow2(s->block_size))
    return fail(FA_ERR_UNSUPPORTED_HEAD_OR_BLOCK_SIZE, "block_size %d must be a power of two >= 16", s->block_size);
  if ((int64_t)s->max_blocks_per_seq * s->block_size > 0x7fffffffLL)
    return fail(FA_ERR_BAD_SHAPE, "a block table of more than 2^31 - 1 tokens is not supported");
  if (s->rotary_dim < 0 || s->rotary_dim % 16 || s->rotary_dim > s->head_size)
    return fail(FA_ERR_BAD_SHAPE, "rotary_dim %d must be a multiple of 16 within head_size %d", s->rotary_dim, s->head_size);
  if (s->rotary_dim > 0 && (s->max_positions <= 0 || (!nothing && !cos_sin)))
    return fail(FA_ERR_NULL_POINTER, "rotary_dim %d needs cos_sin with max_positions > 0 rows", s->rotary_dim);
  if (query && (s->num_heads <= 0)) return fail(FA_ERR_BAD_SHAPE, "num_heads must be positive");
  const int mode = s->kv_scale_mode;
  if (c == FA_KV_CACHE_I8 ? mode != FA_KV_SCALE_BLOCK
                          : mode != FA_KV_SCALE_TENSOR && (c == FA_KV_CACHE_16BIT || mode != FA_KV_SCALE_HEAD))
    return fail(FA_ERR_BAD_SHAPE, "kv_scale_mode %d does not go with cache_dtype %d: integers take block (2), FP8 tensor (0) or "
                                  "head (1), 16-bit pools none (0)", mode, c);
  if (mode != FA_KV_SCALE_TENSOR && !nothing && (!k_scales || !v_scales))
    return fail(FA_ERR_NULL_POINTER, "kv_scale_mode %d needs k_scales and v_scales", mode);
  if (((uintptr_t)k_scales | (uintptr_t)v_scales | (uintptr_t)block_tables | (uintptr_t)query_start | (uintptr_t)context_lens) % 4)
    return fail(FA_ERR_BAD_SHAPE, "k_scales, v_scales, block_tables, query_start and context_lens must be 4-byte aligned");
  const int64_t eb = c == FA_KV_CACHE_16BIT ? 2 : 1;
  if (s->kv_block_stride <= 0 || s->kv_token_stride < s->head_size || s->kv_head_stride < s->head_size)
    return fail(FA_ERR_BAD_SHAPE, "kv strides must be positive and cover one head_size row");
  if ((s->kv_block_stride * eb) % 16 || (s->kv_token_stride * eb) % 16 || (s->kv_head_stride * eb) % 16)
    return fail(FA_ERR_BAD_SHAPE, "kv strides must be multiples of 16 bytes");
  for (int64_t v : {s->key_token_stride, s->key_head_stride, s->value_token_stride, s->value_head_stride,
                    query ? s->query_token_stride : s->head_size, query ? s->query_head_stride : s->head_size,
                    query ? s->query_out_token_stride : s->head_size, query ? s->query_out_head_stride : s->head_size})
    if (v < s->head_size || v % 8) return fail(FA_ERR_BAD_SHAPE, "token and head strides must cover one head_size row and be multiples of 16 bytes");
  if (((uintptr_t)query | (uintptr_t)query_out | (uintptr_t)key | (uintptr_t)value | (uintptr_t)key_cache | (uintptr_t)value_cache |
       (uintptr_t)cos_sin) % 16)
    return fail(FA_ERR_BAD_SHAPE, "query, query_out, key, value, the pools and cos_sin must be 16-byte aligned");
  const int units = s->head_size / 16;
  const int64_t rows_per_token = (query ? s->num_heads : 0) + 2 * (int64_t)s->num_kv_heads;
  if (rows_per_token * units > 0xffffff) return fail(FA_ERR_BAD_SHAPE, "num_heads, num_kv_heads or head_size is too large");
  if (o && o->validate_only) return FA_OK;
  if (o && o->elapsed_us) o->elapsed_us[0] = 0.f;
  if (nothing) return FA_OK;

  KvAppendParams p = {};
  p.b.query_start = query_start;
  p.b.context_lens = context_lens;
  p.b.block_tables = block_tables;
  p.b.num_seqs = s->num_seqs;
  p.b.num_tokens = s->num_tokens;
  p.b.max_blocks_per_seq = s->max_blocks_per_seq;
  p.b.block_shift = ilog2(s->block_size);
  p.b.max_block_id = s->num_pool_blocks - 1;
  p.query = reinterpret_cast<const char *>(query);
  p.query_out = reinterpret_cast<char *>(query_out);
  p.key = reinterpret_cast<const char *>(key);
  p.value = reinterpret_cast<const char *>(value);
  p.key_cache = reinterpret_cast<char *>(key_cache);
  p.value_cache = reinterpret_cast<char *>(value_cache);
  p.cos_sin = s->rotary_dim > 0 ? cos_sin : nullptr;
  p.k_scales = mode != FA_KV_SCALE_TENSOR ? k_scales : nullptr;
  p.v_scales = mode != FA_KV_SCALE_TENSOR ? v_scales : nullptr;
  p.scale_block_pitch = s->num_kv_heads;
  p.inv_scale = 1.0f / (s->fp8_scale != 0.f ? s->fp8_scale : 1.0f);
  p.max_positions = s->max_positions;
  p.rotary = s->rotary_dim;
  p.num_heads = s->num_heads;
  p.num_kv_heads = s->num_kv_heads;
  p.block_size = s->block_size;
  p.q_token_bytes = s->query_token_stride * 2;
  p.q_head_bytes = s->query_head_stride * 2;
  p.qo_token_bytes = s->query_out_token_stride * 2;
  p.qo_head_bytes = s->query_out_head_stride * 2;
  p.src_token_bytes = s->key_token_stride * 2;
  p.src_head_bytes = s->key_head_stride * 2;
  p.val_token_bytes = s->value_token_stride * 2;
  p.val_head_bytes = s->value_head_stride * 2;
  p.kv_block_bytes = s->kv_block_stride * eb;
  p.kv_token_bytes = s->kv_token_stride * eb;
  p.kv_head_bytes = s->kv_head_stride * eb;
  p.pairs_per_row = units;

  const hipStream_t stream = o ? reinterpret_cast<hipStream_t>(o->stream) : nullptr;
  KernelTimer timer(o && o->elapsed_us, stream);
  const bool bf16 = s->src_dtype == FA_DTYPE_BF16, inter = s->interleaved != 0;
  const int64_t T = s->num_tokens;
  auto groups_of = [&](int64_t rows) {  // work-groups for `rows` rows of every token, and how they are cut
    p.units_per_token = (int32_t)(rows * units);
    const int64_t all = T * p.units_per_token;
    const int per_thread = all >= 256 * 4 * 2048 ? 4 : 1;
    p.tokens_per_group = (int32_t)std::min<int64_t>(kAppendMaxTokens, std::max<int64_t>(1, 256 * per_thread / std::max(1, p.units_per_token)));
    return (T + p.tokens_per_group - 1) / p.tokens_per_group;
  };
  int64_t groups = 0;
#define FA_APPEND_LAUNCH(KERNEL) FA_HIP_CHECK(timer.launch(KERNEL, dim3((unsigned)groups), dim3(256), 0, p))
#define FA_APPEND_TYPES(NAME, ...)                                                              \
  do {                                                                                          \
    if (bf16) {                                                                                 \
      if (inter) FA_APPEND_LAUNCH((NAME<BF16, __VA_ARGS__ true>));                              \
      else FA_APPEND_LAUNCH((NAME<BF16, __VA_ARGS__ false>));                                   \
    } else {                                                                                    \
      if (inter) FA_APPEND_LAUNCH((NAME<F16, __VA_ARGS__ true>));                               \
      else FA_APPEND_LAUNCH((NAME<F16, __VA_ARGS__ false>));                                    \
    }                                                                                           \
  } while (0)
#define FA_COMMA ,
  if (c == FA_KV_CACHE_I8) {
    const int64_t query_groups = query ? groups_of(s->num_heads) : 0;
    // blocks of few tokens leave nothing for more than one wavefront to do
    const int batch = 2 * std::max(1, 64 / units);
    p.team = s->block_size <= batch ? 1 : s->block_size <= 2 * batch ? 2 : 4;
    // A work-group for each token finds its owner at once, and most find none where sequences bring many tokens; one for a block's
    // worth of tokens goes through its owners one after the other.  us of the two (8 kv heads of 128): single tokens of 512
    // sequences, blocks of 16: 11 and 29, of 1536 29 and 35, of 2048 39 and 35; blocks of 64: 26 and 100, 80 and 108, 113 and
    // 108.  500 times 2: 18 and 18 (blocks of 64: 46 and 55), 700 times 2 24 and 21 (65 and 59), 250 times 4 17 and 13 (39 and 33); prompts
    // of 256 tokens 9 and 9 (10 and 11), of 1000 16 and 9 (30 and 11), three of 4000 118 and 21 (315 and 30).
    p.window = T <= std::min<int64_t>(512 + (int64_t)s->num_seqs, 1536) ? 1 : std::min(s->block_size, kAppendMaxTokens);
    const int teams = 4 / p.team;
    const int64_t unit_groups = (2 * (int64_t)s->num_kv_heads + teams - 1) / teams;
    const int64_t kv_groups = (T + p.window - 1) / p.window * unit_groups;
    groups = kv_groups + query_groups;
    if (groups > 0x7fffffff) return fail(FA_ERR_BAD_SHAPE, "%lld work-groups exceed the grid limit 2^31 - 1", (long long)groups);
    p.kv_groups = (int32_t)kv_groups;
    FA_APPEND_TYPES(kv_cache_append_scaled_kernel, );
  } else {
    groups = groups_of(rows_per_token);
    if (c == FA_KV_CACHE_16BIT) FA_APPEND_TYPES(kv_cache_append_kernel, kKv16 FA_COMMA);
    else if (c == FA_KV_CACHE_E4M3) FA_APPEND_TYPES(kv_cache_append_kernel, kKvE4M3 FA_COMMA);
    else FA_APPEND_TYPES(kv_cache_append_kernel, kKvE5M2 FA_COMMA);
  }
#undef FA_COMMA
#undef FA_APPEND_TYPES
#undef FA_APPEND_LAUNCH
  if (o && o->elapsed_us) FA_HIP_CHECK(timer.read(0, &o->elapsed_us[0]));
  return FA_OK;
}

}  // namespace fa
