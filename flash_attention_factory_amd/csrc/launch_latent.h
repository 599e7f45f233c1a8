// Host launchers of latent attention (declared in include/fa_latent.h): argument checks, tile sizes and work-group counts, workspace.
#pragma once

#include <algorithm>

#include "../../include/fa_latent.h"
#include "latent_expanded_kernel.h"
#include "launch_common.h"

namespace fa {

inline bool is_16bit_dtype(int32_t t) { return t == FA_DTYPE_F16 || t == FA_DTYPE_BF16; }

// What every entry over a pool asks of it.
inline fa_status check_latent_pool(int32_t latent_dim, int32_t rope_dim, int32_t block_size, int32_t max_blocks_per_seq, int32_t num_pool_blocks,
                                   int32_t cache_dtype, int64_t block_stride, int64_t token_stride) {
  if ((latent_dim != 256 && latent_dim != 512) || rope_dim != kLatentRope || block_size < 16 || !is_pow2(block_size))
    return fail(FA_ERR_UNSUPPORTED_HEAD_OR_BLOCK_SIZE,
                "Unsupported head size or block size (latent_dim %d must be 256 or 512, rope_dim %d 64, block_size %d a power of two >= 16)",
                latent_dim, rope_dim, block_size);
  if (max_blocks_per_seq <= 0 || num_pool_blocks <= 0) return fail(FA_ERR_BAD_SHAPE, "max_blocks_per_seq and num_pool_blocks must be positive");
  if ((int64_t)max_blocks_per_seq * block_size > 0x3fffffffLL) return fail(FA_ERR_BAD_SHAPE, "a block table of 2^30 tokens or more is not supported");
  if (cache_dtype != FA_KV_CACHE_16BIT && cache_dtype != FA_KV_CACHE_E4M3)
    return fail(FA_ERR_UNSUPPORTED_DTYPE, "cache_dtype %d is neither 16-bit (0) nor E4M3 (2)", cache_dtype);
  const int64_t eb = cache_dtype == FA_KV_CACHE_16BIT ? 2 : 1;
  if (block_stride <= 0 || token_stride < latent_dim + rope_dim) return fail(FA_ERR_BAD_SHAPE, "pool strides must be positive and cover one row");
  if ((block_stride * eb) % 16 || (token_stride * eb) % 16) return fail(FA_ERR_BAD_SHAPE, "pool strides must be multiples of 16 bytes");
  if (block_stride > 0x7fffffffLL || token_stride > 0x7ffffffLL) return fail(FA_ERR_BAD_SHAPE, "pool strides are too large");
  return FA_OK;
}

// Strides of rows of `row` 16-bit elements.
inline fa_status check_row_strides(std::initializer_list<int64_t> strides, int64_t row, const char *name) {
  for (int64_t v : strides)
    if (v < row || v % 8) return fail(FA_ERR_BAD_SHAPE, "%s strides must cover one row of %lld elements and be multiples of 16 bytes", name, (long long)row);
  return FA_OK;
}
inline bool aligned_to(std::initializer_list<const void *> pointers, uintptr_t bytes) {
  uintptr_t all = 0;
  for (const void *p : pointers) all |= (uintptr_t)p;
  return all % bytes == 0;
}

inline RaggedBatch latent_batch(const int32_t *block_tables, const int32_t *query_start, const int32_t *context_lens, int32_t num_seqs,
                                int32_t num_tokens, int32_t max_blocks_per_seq, int32_t block_size, int32_t num_pool_blocks) {
  RaggedBatch b = {};
  b.query_start = query_start;
  b.context_lens = context_lens;
  b.block_tables = block_tables;
  b.num_seqs = num_seqs;
  b.num_tokens = num_tokens;
  b.max_blocks_per_seq = max_blocks_per_seq;
  b.block_shift = ilog2(block_size);
  b.max_block_id = num_pool_blocks - 1;
  return b;
}

inline fa_status launch_latent_cache_append(const void *latent, const void *rope_key, void *cache, const float *norm_weight, const float *cos_sin,
                                            const void *query_rope, void *query_rope_out, float *scales, const int32_t *block_tables,
                                            const int32_t *query_start, const int32_t *context_lens, const fa_latent_append_shape *s,
                                            const fa_paged_attention_options *o) {
  if (s->num_seqs < 0 || s->num_tokens < 0 || s->max_positions < 0)
    return fail(FA_ERR_BAD_SHAPE, "num_seqs, num_tokens and max_positions must be >= 0");
  fa_status st = check_latent_pool(s->latent_dim, s->rope_dim, s->block_size, s->max_blocks_per_seq, s->num_pool_blocks, s->cache_dtype,
                                   s->block_stride, s->token_stride);
  if (st != FA_OK) return st;
  const bool nothing = s->num_tokens == 0 || s->num_seqs == 0, kv8 = s->cache_dtype == FA_KV_CACHE_E4M3;
  if (!nothing && (!latent || !rope_key || !cache || !block_tables || !query_start || !context_lens))
    return fail(FA_ERR_NULL_POINTER, "latent, rope_key, cache, block_tables, query_start and context_lens must all be non-NULL");
  if (!nothing && (query_rope == nullptr) != (query_rope_out == nullptr)) return fail(FA_ERR_NULL_POINTER, "query_rope and query_rope_out come together");
  if (!nothing && kv8 && !scales) return fail(FA_ERR_NULL_POINTER, "E4M3 pools need scales");
  if (!nothing && s->max_positions > 0 && !cos_sin) return fail(FA_ERR_NULL_POINTER, "max_positions %d needs cos_sin", s->max_positions);
  if (!is_16bit_dtype(s->src_dtype)) return fail(FA_ERR_UNSUPPORTED_DTYPE, "src_dtype %d is neither fp16 (0) nor bf16 (1)", s->src_dtype);
  if ((st = check_row_strides({s->latent_token_stride}, s->latent_dim, "latent")) != FA_OK) return st;
  if ((st = check_row_strides({s->rope_key_token_stride}, s->rope_dim, "rope_key")) != FA_OK) return st;
  if (query_rope) {
    if (s->num_heads <= 0 || s->num_heads > 4096) return fail(FA_ERR_BAD_SHAPE, "num_heads must be positive, at most 4096");
    if ((st = check_row_strides({s->query_token_stride, s->query_head_stride, s->query_out_token_stride, s->query_out_head_stride}, s->rope_dim,
                                "query")) != FA_OK)
      return st;
  }
  if (!aligned_to({latent, rope_key, cache, norm_weight, cos_sin, query_rope, query_rope_out}, 16))
    return fail(FA_ERR_BAD_SHAPE, "latent, rope_key, cache, norm_weight, cos_sin, query_rope and query_rope_out must be 16-byte aligned");
  if (!aligned_to({scales, block_tables, query_start, context_lens}, 4))
    return fail(FA_ERR_BAD_SHAPE, "scales, block_tables, query_start and context_lens must be 4-byte aligned");
  if (!(s->norm_eps >= 0.f)) return fail(FA_ERR_BAD_SHAPE, "norm_eps must be >= 0");
  if (o && o->validate_only) return FA_OK;
  if (o && o->elapsed_us) o->elapsed_us[0] = 0.f;
  if (nothing) return FA_OK;

  const int64_t eb = kv8 ? 1 : 2;
  LatentAppendParams p = {};
  p.a.b = latent_batch(block_tables, query_start, context_lens, s->num_seqs, s->num_tokens, s->max_blocks_per_seq, s->block_size, s->num_pool_blocks);
  p.a.query = reinterpret_cast<const char *>(query_rope);
  p.a.query_out = reinterpret_cast<char *>(query_rope_out);
  p.a.key_cache = reinterpret_cast<char *>(cache);
  p.a.cos_sin = s->max_positions > 0 ? cos_sin : nullptr;
  p.a.max_positions = s->max_positions;
  p.a.rotary = kLatentRope;
  p.a.num_heads = s->num_heads;
  p.a.q_token_bytes = s->query_token_stride * 2;
  p.a.q_head_bytes = s->query_head_stride * 2;
  p.a.qo_token_bytes = s->query_out_token_stride * 2;
  p.a.qo_head_bytes = s->query_out_head_stride * 2;
  p.a.kv_block_bytes = s->block_stride * eb;
  p.a.kv_token_bytes = s->token_stride * eb;
  p.a.pairs_per_row = kLatentRope / 16;
  p.latent = reinterpret_cast<const char *>(latent);
  p.rope_key = reinterpret_cast<const char *>(rope_key);
  p.latent_token_bytes = s->latent_token_stride * 2;
  p.rope_key_token_bytes = s->rope_key_token_stride * 2;
  p.norm_weight = norm_weight;
  p.norm_eps = s->norm_eps;
  p.scales = scales;
  const int64_t T = s->num_tokens;
  p.row_groups = (int32_t)((T + 3) / 4);
  int64_t groups = p.row_groups;
  if (query_rope) {
    p.a.units_per_token = s->num_heads * p.a.pairs_per_row;
    const int per_thread = T * p.a.units_per_token >= 256 * 4 * 2048 ? 4 : 1;
    p.a.tokens_per_group = (int32_t)std::min<int64_t>(kAppendMaxTokens, std::max<int64_t>(1, 256 * per_thread / p.a.units_per_token));
    groups += (T + p.a.tokens_per_group - 1) / p.a.tokens_per_group;
  }
  if (groups > 0x7fffffff) return fail(FA_ERR_BAD_SHAPE, "%lld work-groups exceed the grid limit 2^31 - 1", (long long)groups);
  KernelTimer timer(o && o->elapsed_us, o ? reinterpret_cast<hipStream_t>(o->stream) : nullptr);
  const auto launch = [&](auto dim, auto type, auto bytes, auto inter) {
    return timer.launch(latent_cache_append_kernel<decltype(dim)::value, decltype(type), decltype(bytes)::value, decltype(inter)::value>,
                        dim3((unsigned)groups), dim3(256), 0, p);
  };
  const auto of_dim = [&](auto type, auto bytes, auto inter) {
    return s->latent_dim == 512 ? launch(std::integral_constant<int, 512>{}, type, bytes, inter) : launch(std::integral_constant<int, 256>{}, type, bytes, inter);
  };
  const auto of_pool = [&](auto type, auto inter) { return kv8 ? of_dim(type, std::true_type{}, inter) : of_dim(type, std::false_type{}, inter); };
  const auto of_type = [&](auto inter) { return s->src_dtype == FA_DTYPE_BF16 ? of_pool(BF16{}, inter) : of_pool(F16{}, inter); };
  FA_HIP_CHECK(s->interleaved ? of_type(std::true_type{}) : of_type(std::false_type{}));
  if (o && o->elapsed_us) FA_HIP_CHECK(timer.read(0, &o->elapsed_us[0]));
  return FA_OK;
}

inline fa_status launch_latent_cache_gather(void *out, const void *cache, const float *scales, const int32_t *block_tables, const int32_t *row_start,
                                            const int32_t *first_keys, const fa_latent_gather_shape *s, const fa_paged_attention_options *o) {
  if (s->num_seqs < 0 || s->num_rows < 0) return fail(FA_ERR_BAD_SHAPE, "num_seqs and num_rows must be >= 0");
  fa_status st = check_latent_pool(s->latent_dim, s->rope_dim, s->block_size, s->max_blocks_per_seq, s->num_pool_blocks, s->cache_dtype,
                                   s->block_stride, s->token_stride);
  if (st != FA_OK) return st;
  const bool nothing = s->num_rows == 0 || s->num_seqs == 0, kv8 = s->cache_dtype == FA_KV_CACHE_E4M3;
  if (!nothing && (!out || !cache || !block_tables || !row_start)) return fail(FA_ERR_NULL_POINTER, "out, cache, block_tables and row_start must all be non-NULL");
  if (!nothing && kv8 && !scales) return fail(FA_ERR_NULL_POINTER, "E4M3 pools need scales");
  if (!is_16bit_dtype(s->out_dtype)) return fail(FA_ERR_UNSUPPORTED_DTYPE, "out_dtype %d is neither fp16 (0) nor bf16 (1)", s->out_dtype);
  if ((st = check_row_strides({s->out_stride}, s->latent_dim + s->rope_dim, "out")) != FA_OK) return st;
  if (!aligned_to({out, cache}, 16)) return fail(FA_ERR_BAD_SHAPE, "out and cache must be 16-byte aligned");
  if (!aligned_to({scales, block_tables, row_start, first_keys}, 4))
    return fail(FA_ERR_BAD_SHAPE, "scales, block_tables, row_start and first_keys must be 4-byte aligned");
  if (o && o->validate_only) return FA_OK;
  if (o && o->elapsed_us) o->elapsed_us[0] = 0.f;
  if (nothing) return FA_OK;

  LatentGatherParams p = {};
  p.b = latent_batch(block_tables, row_start, nullptr, s->num_seqs, s->num_rows, s->max_blocks_per_seq, s->block_size, s->num_pool_blocks);
  p.cache = reinterpret_cast<const char *>(cache);
  p.scales = scales;
  p.first_keys = first_keys;
  p.out = reinterpret_cast<char *>(out);
  p.block_bytes = s->block_stride * (kv8 ? 1 : 2);
  p.token_bytes = s->token_stride * (kv8 ? 1 : 2);
  p.out_bytes = s->out_stride * 2;
  // (141 000 FP8 rows, from memory: 16 rows a work-group 57.0 us, 32 59.4, 64 64.8; few rows: more work-groups, so that all of them start at once)
  p.rows_per_group = s->num_rows >= 16384 ? 16 : 8;
  const unsigned groups = (unsigned)((s->num_rows + (int64_t)p.rows_per_group - 1) / p.rows_per_group);
  KernelTimer timer(o && o->elapsed_us, o ? reinterpret_cast<hipStream_t>(o->stream) : nullptr);
  const auto launch = [&](auto dim, auto type, auto bytes) {
    return timer.launch(latent_cache_gather_kernel<decltype(dim)::value, decltype(type), decltype(bytes)::value>, dim3(groups), dim3(256), 0, p);
  };
  const auto of_dim = [&](auto type, auto bytes) {
    return s->latent_dim == 512 ? launch(std::integral_constant<int, 512>{}, type, bytes) : launch(std::integral_constant<int, 256>{}, type, bytes);
  };
  if (!kv8) FA_HIP_CHECK(of_dim(F16{}, std::false_type{}));  // (bits are copied, whichever 16-bit type they are of)
  else if (s->out_dtype == FA_DTYPE_BF16) FA_HIP_CHECK(of_dim(BF16{}, std::true_type{}));
  else FA_HIP_CHECK(of_dim(F16{}, std::true_type{}));
  if (o && o->elapsed_us) FA_HIP_CHECK(timer.read(0, &o->elapsed_us[0]));
  return FA_OK;
}

// ---- absorbed attention ----

struct LatentPlan {
  int rows;             // M, of a tile: 32, 64 or 128
  int64_t tile_bound;   // tiles, at most
  int team;             // tiles side by side on the line
  int groups;           // shares of the line, for `team` work-groups each; 0: a work-group for each tile
  int64_t part_o, part_ml, joins, bytes;
};

inline fa_status check_latent_attention_shape(const fa_latent_attention_shape *s) {
  if (s->num_seqs < 0 || s->num_tokens < 0 || s->num_heads <= 0 || s->max_query_len <= 0 || s->max_context_len < 0)
    return fail(FA_ERR_BAD_SHAPE, "num_seqs, num_tokens and max_context_len must be >= 0; num_heads and max_query_len positive");
  const fa_status st = check_latent_pool(s->latent_dim, s->rope_dim, s->block_size, s->max_blocks_per_seq, s->num_pool_blocks, s->cache_dtype,
                                         s->block_stride, s->token_stride);
  if (st != FA_OK) return st;
  if (!is_16bit_dtype(s->q_dtype)) return fail(FA_ERR_UNSUPPORTED_DTYPE, "q_dtype %d is neither fp16 (0) nor bf16 (1)", s->q_dtype);
  if (((int64_t)s->num_tokens + s->num_seqs) * s->num_heads > 0x3fffffffLL) return fail(FA_ERR_BAD_SHAPE, "num_tokens x num_heads is too large");
  // the line of tiles is as long as the sum of their steps, and cut at products with the work-groups' numbers
  const int64_t steps = (int64_t)s->max_blocks_per_seq * s->block_size / LatentSteps<false, 32>::kKeys + 8;
  if (((int64_t)s->num_tokens * s->num_heads / 32 + s->num_seqs) * steps > (1LL << 41))
    return fail(FA_ERR_BAD_SHAPE, "num_tokens x num_heads x keys is too large");
  return FA_OK;
}

// Up to as many keys tiles are not cut.
constexpr int kLatentWhole = 256;

inline LatentPlan latent_plan(const fa_latent_attention_shape &s, int cus) {
  LatentPlan r = {};
  r.team = 1;
  const int64_t T = s.num_tokens, S = s.num_seqs, H = s.num_heads;
  if (T == 0 || S == 0) return r;
  const int64_t most = std::min<int64_t>(s.max_query_len, T), table = (int64_t)s.max_blocks_per_seq * s.block_size;
  const int64_t keys = s.max_context_len > 0 ? std::min<int64_t>(s.max_context_len, table) : table;
  auto tiles_of = [&](int64_t rows) { return std::min(S * ((most * H + rows - 1) / rows), T * H / rows + S); };
  auto passes = [&](int64_t rows) { return (tiles_of(rows) + cus - 1) / cus; };
  // Tiles of 128 rows go through the keys in less time for each row (a round of 32 keys 1.9 us, of 64 rows 1.3 us).  But what is left of
  // cut ones to be joined is twice as large (256 KiB for each work-group to write and to read), and so is what one alone costs at its
  // start and end (64 heads, 13 sequences of 301 to 9000 FP8 keys, 2 to 6 tokens: 57 us with 128 rows, 53 us with 64; 128 heads, 64
  // sequences of 512 to 16384 keys: 126 us and 136 us).  Cut tiles pay from about 16 rounds for each compute unit on; of the longest
  // context's rounds, four times as many.  Whole ones (short contexts) pay where they save a pass over the compute units.
  // The host knows the longest context only, and the four fit contexts that are spread.  Where they are equal, 64 rows are taken for longer
  // than they pay: 128 heads, us with 64 and 128 rows, 16-bit pools 67 and 77 at 16 rounds, 113 and 116 at 32, 213 and 188 at 64 (where the
  // rule changes over); FP8 57 and 56 at 8, 81 and 76 at 16, 131 and 110 at 32.
  // One height serves the whole batch, by its longest piece: 16 heads, 128 sequences of 512 to 16384 keys with a token each beside a piece of
  // 64 tokens take 157 us (16-bit; as two calls 179), with FP8 pools, whose 32-row tiles are the faster ones, 159 us (as two calls 121).
  bool tall = most * H > 64;
  if (tall && keys > kLatentWhole) tall = (T * H / 128) * (keys / 32) >= 64 * cus;
  else if (tall) tall = passes(128) * (11 + 1.9 * (keys / 32 + 1)) < passes(64) * (8 + 1.3 * (keys / 32 + 1));
  r.rows = most * H <= 32 ? 32 : tall ? 128 : 64;
  const int64_t each = (most * H + r.rows - 1) / r.rows;
  r.tile_bound = tiles_of(r.rows);
  if (keys > kLatentWhole) {
    const bool equal = S == 1 || T == S * most;  // every sequence brings `most` tokens
    r.team = !equal ? 1 : each % 4 == 0 ? 4 : each % 2 == 0 ? 2 : 1;
    r.groups = std::max(8, cus / r.team / 8 * 8);  // (an eighth of the shares for each XCC)
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
      const int64_t here = at;
      at += (bytes + 255) / 256 * 256;
      return here;
    };
    r.part_o = take(2 * (int64_t)r.groups * r.team * r.rows * s.latent_dim * 4);
    r.part_ml = take(2 * (int64_t)r.groups * r.team * 2 * r.rows * 4);
    r.joins = take((int64_t)r.groups * r.team * sizeof(LatentJoin));
    r.bytes = at;
  }
  return r;
}

template <int L, typename OT, bool KV8, int M>
inline fa_status launch_latent_tiles(const LatentParams &p, const LatentPlan &plan, KernelTimer &timer, float *us) {
  const dim3 grid((unsigned)(plan.groups > 0 ? plan.groups * plan.team : plan.tile_bound));
  FA_HIP_CHECK(timer.launch(latent_absorbed_kernel<L, OT, KV8, M>, grid, dim3(512), 0, p));
  if (us) FA_HIP_CHECK(timer.accumulate(0, us));
  if (plan.groups > 0) {
    // tiles that are cut: no more than there are, and than the shares' ends
    const int64_t cut = std::min<int64_t>(plan.tile_bound, (int64_t)(plan.groups - 1) * plan.team);
    FA_HIP_CHECK(timer.launch(latent_absorbed_join_kernel<L, OT, KV8, M>, dim3((unsigned)cut, M * L / 1024), dim3(256), 0, p));
    if (us) FA_HIP_CHECK(timer.accumulate(0, us));
  }
  return FA_OK;
}

inline fa_status launch_latent_attention(void *out, const void *query_latent, const void *query_rope, const void *cache, const float *scales,
                                         const int32_t *block_tables, const int32_t *query_start, const int32_t *context_lens, float scale,
                                         void *workspace, int64_t workspace_bytes, const fa_latent_attention_shape *s,
                                         const fa_paged_attention_options *o) {
  fa_status st = check_latent_attention_shape(s);
  if (st != FA_OK) return st;
  const bool nothing = s->num_tokens == 0 || s->num_seqs == 0, kv8 = s->cache_dtype == FA_KV_CACHE_E4M3;
  if (!nothing && (!out || !query_latent || !query_rope || !cache || !block_tables || !query_start || !context_lens))
    return fail(FA_ERR_NULL_POINTER, "out, query_latent, query_rope, cache, block_tables, query_start and context_lens must all be non-NULL");
  if (!nothing && kv8 && !scales) return fail(FA_ERR_NULL_POINTER, "E4M3 pools need scales");
  if ((st = check_row_strides({s->query_latent_token_stride, s->query_latent_head_stride, s->out_token_stride, s->out_head_stride}, s->latent_dim,
                              "query_latent and out")) != FA_OK)
    return st;
  if ((st = check_row_strides({s->query_rope_token_stride, s->query_rope_head_stride}, s->rope_dim, "query_rope")) != FA_OK) return st;
  if (!aligned_to({out, query_latent, query_rope, cache, workspace}, 16))
    return fail(FA_ERR_BAD_SHAPE, "out, query_latent, query_rope, cache and workspace must be 16-byte aligned");
  if (!aligned_to({scales, block_tables, query_start, context_lens}, 4))
    return fail(FA_ERR_BAD_SHAPE, "scales, block_tables, query_start and context_lens must be 4-byte aligned");
  if (!(scale - scale == 0.f)) return fail(FA_ERR_BAD_SHAPE, "scale must be finite");
  if (o && o->validate_only) return FA_OK;
  if (o && o->elapsed_us) o->elapsed_us[0] = 0.f;
  if (nothing) return FA_OK;
  int cus = 0;
  FA_HIP_CHECK(compute_units_of_current_device(&cus));
  const LatentPlan plan = latent_plan(*s, cus);
  if (workspace_bytes < plan.bytes || (plan.bytes > 0 && !workspace))
    return fail(FA_ERR_SCRATCH_TOO_SMALL, "the call works in %lld bytes of workspace, %lld were given", (long long)plan.bytes,
                (long long)(workspace ? workspace_bytes : 0));

  const int64_t eb = kv8 ? 1 : 2;
  LatentParams p = {};
  p.b = latent_batch(block_tables, query_start, context_lens, s->num_seqs, s->num_tokens, s->max_blocks_per_seq, s->block_size, s->num_pool_blocks);
  p.cache = reinterpret_cast<const char *>(cache);
  p.scales = scales;
  p.block_bytes = (uint32_t)(s->block_stride * eb);
  p.token_bytes = (uint32_t)(s->token_stride * eb);
  p.query_latent = reinterpret_cast<const char *>(query_latent);
  p.query_rope = reinterpret_cast<const char *>(query_rope);
  p.ql_token_bytes = s->query_latent_token_stride * 2;
  p.ql_head_bytes = s->query_latent_head_stride * 2;
  p.qr_token_bytes = s->query_rope_token_stride * 2;
  p.qr_head_bytes = s->query_rope_head_stride * 2;
  p.out = reinterpret_cast<char *>(out);
  p.out_token_bytes = s->out_token_stride * 2;
  p.out_head_bytes = s->out_head_stride * 2;
  p.num_heads = s->num_heads;
  p.max_query_len = s->max_query_len;
  p.score_scale_log2 = std::abs(scale) * kLog2e;
  p.query_flip = scale < 0.f ? 0x80008000u : 0u;
  p.groups = plan.groups;
  p.team = plan.team;
  p.part_o = reinterpret_cast<float *>(reinterpret_cast<char *>(workspace) + plan.part_o);
  p.part_ml = reinterpret_cast<float *>(reinterpret_cast<char *>(workspace) + plan.part_ml);
  p.joins = reinterpret_cast<LatentJoin *>(reinterpret_cast<char *>(workspace) + plan.joins);
  float *us = o ? o->elapsed_us : nullptr;
  KernelTimer timer(us != nullptr, o ? reinterpret_cast<hipStream_t>(o->stream) : nullptr);
  const auto of_rows = [&](auto dim, auto type, auto bytes) {
    constexpr int kDim = decltype(dim)::value;
    constexpr bool kBytes = decltype(bytes)::value;
    using Type = decltype(type);
    return plan.rows == 32   ? launch_latent_tiles<kDim, Type, kBytes, 32>(p, plan, timer, us)
           : plan.rows == 64 ? launch_latent_tiles<kDim, Type, kBytes, 64>(p, plan, timer, us)
                             : launch_latent_tiles<kDim, Type, kBytes, 128>(p, plan, timer, us);
  };
  const auto of_dim = [&](auto type, auto bytes) {
    return s->latent_dim == 512 ? of_rows(std::integral_constant<int, 512>{}, type, bytes) : of_rows(std::integral_constant<int, 256>{}, type, bytes);
  };
  const auto of_type = [&](auto bytes) { return s->q_dtype == FA_DTYPE_BF16 ? of_dim(BF16{}, bytes) : of_dim(F16{}, bytes); };
  return kv8 ? of_type(std::true_type{}) : of_type(std::false_type{});
}

// ---- expanded attention ----

struct ExpandedPlan {
  int wavefronts;       // of a work-group
  int64_t tile_bound;   // tiles of one head, at most
  int groups;           // work-groups that share the line of tiles; 0: a work-group for each tile
  int64_t tile_o, tile_ml, bytes;
};

inline fa_status check_latent_expanded_shape(const fa_latent_expanded_shape *s) {
  if (s->num_seqs < 0 || s->num_tokens < 0 || s->num_keys < 0 || s->num_heads <= 0 || s->max_query_len <= 0 || s->max_key_len < 0)
    return fail(FA_ERR_BAD_SHAPE, "num_seqs, num_tokens, num_keys and max_key_len must be >= 0; num_heads and max_query_len positive");
  if ((s->head_size != 64 && s->head_size != 128) || s->rope_dim != kLatentRope)
    return fail(FA_ERR_UNSUPPORTED_HEAD_OR_BLOCK_SIZE, "Unsupported head size or block size (head_size %d must be 64 or 128, rope_dim %d 64)", s->head_size,
                s->rope_dim);
  if (!is_16bit_dtype(s->dtype)) return fail(FA_ERR_UNSUPPORTED_DTYPE, "dtype %d is neither fp16 (0) nor bf16 (1)", s->dtype);
  if (s->num_keys > 0x3fffffff || ((int64_t)s->num_tokens / 32 + s->num_seqs) * s->num_heads > 0x3fffffffLL)
    return fail(FA_ERR_BAD_SHAPE, "num_keys or num_tokens x num_heads is too large");
  if (((int64_t)s->num_tokens / 32 + s->num_seqs) * s->num_heads * ((int64_t)s->num_keys + 1024) > (1LL << 41))
    return fail(FA_ERR_BAD_SHAPE, "num_tokens x num_heads x num_keys is too large");
  return FA_OK;
}

inline ExpandedPlan expanded_plan(const fa_latent_expanded_shape &s, int cus) {
  ExpandedPlan r = {};
  const int64_t T = s.num_tokens, S = s.num_seqs, H = s.num_heads;
  if (T == 0 || S == 0) return r;
  const int64_t most = std::min<int64_t>(s.max_query_len, T);
  const int64_t keys = s.max_key_len > 0 ? std::min<int64_t>(s.max_key_len, s.num_keys) : s.num_keys;
  r.wavefronts = most <= 128 || keys <= 1536 ? 4 : 8;
  const int64_t rows = r.wavefronts * 32, each = (most + rows - 1) / rows;
  r.tile_bound = std::min(S * each, T / rows + S);
  // Tiles for each compute unit: from two on, a work-group each, longest first, keeps them all busy.  With fewer, the longest
  // tile (or two one after the other) leaves compute units idle for so many keys; shares of a line do not, but cost a second
  // kernel and their bookkeeping, about what 20 steps take.
  const double x = (double)(r.tile_bound * H) / cus, mean = std::max<double>((double)keys - most / 2, 0);
  if (x < 2 && std::max<double>((double)keys, x > 1 ? 2 * mean : mean) - x * mean > 20 * kTileKeys) {
    const int64_t resident = (int64_t)cus * (r.wavefronts == 4 ? 2 : 1);
    r.groups = (int)std::max<int64_t>(8, resident / 8 * 8);  // (an eighth of the shares for each XCC)
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
      const int64_t here = at;
      at += (bytes + 255) / 256 * 256;
      return here;
    };
    r.tile_o = take(2 * (int64_t)r.groups * r.wavefronts * s.head_size * 32 * 4);
    r.tile_ml = take(2 * (int64_t)r.groups * r.wavefronts * 128 * 4);
    r.bytes = at;
  }
  return r;
}

template <int D, typename OT, int NW>
inline fa_status launch_expanded_tiles(const ExpandedParams &p, const ExpandedPlan &plan, KernelTimer &timer, float *us) {
  const dim3 grid((unsigned)(plan.groups > 0 ? plan.groups : plan.tile_bound * p.num_kv_heads)), block(NW * 64);
  FA_HIP_CHECK(plan.groups > 0 ? timer.launch(latent_expanded_kernel<D, OT, NW, true>, grid, block, 0, p)
                               : timer.launch(latent_expanded_kernel<D, OT, NW, false>, grid, block, 0, p));
  if (us) FA_HIP_CHECK(timer.accumulate(0, us));
  if (plan.groups > 1) {
    FA_HIP_CHECK(timer.launch(latent_expanded_join_kernel<D, OT, NW>, dim3((unsigned)(plan.groups - 1)), block, 0, p));
    if (us) FA_HIP_CHECK(timer.accumulate(0, us));
  }
  return FA_OK;
}

inline fa_status launch_latent_expanded(void *out, const void *query, const void *key, const void *rope_key, const void *value,
                                        const int32_t *query_start, const int32_t *key_start, float scale, void *workspace,
                                        int64_t workspace_bytes, const fa_latent_expanded_shape *s, const fa_paged_attention_options *o) {
  fa_status st = check_latent_expanded_shape(s);
  if (st != FA_OK) return st;
  const bool nothing = s->num_tokens == 0 || s->num_seqs == 0;
  if (!nothing && (!out || !query || !query_start || !key_start || (s->num_keys > 0 && (!key || !rope_key || !value))))
    return fail(FA_ERR_NULL_POINTER, "out, query, key, rope_key, value, query_start and key_start must all be non-NULL");
  if ((st = check_row_strides({s->query_token_stride, s->query_head_stride}, s->head_size + s->rope_dim, "query")) != FA_OK) return st;
  if ((st = check_row_strides({s->key_token_stride, s->key_head_stride, s->value_token_stride, s->value_head_stride, s->out_token_stride, s->out_head_stride},
                              s->head_size, "key, value and out")) != FA_OK)
    return st;
  if ((st = check_row_strides({s->rope_key_token_stride}, s->rope_dim, "rope_key")) != FA_OK) return st;
  for (int64_t v : {s->key_token_stride, s->value_token_stride, s->rope_key_token_stride})
    if (v > 0x3ffffffLL) return fail(FA_ERR_BAD_SHAPE, "token strides of key, value and rope_key must be under 2^26 elements");
  if (!aligned_to({out, query, key, rope_key, value, workspace}, 16))
    return fail(FA_ERR_BAD_SHAPE, "out, query, key, rope_key, value and workspace must be 16-byte aligned");
  if (!aligned_to({query_start, key_start}, 4)) return fail(FA_ERR_BAD_SHAPE, "query_start and key_start must be 4-byte aligned");
  if (!(scale - scale == 0.f)) return fail(FA_ERR_BAD_SHAPE, "scale must be finite");
  if (o && o->validate_only) return FA_OK;
  if (o && o->elapsed_us) o->elapsed_us[0] = 0.f;
  if (nothing) return FA_OK;
  int cus = 0;
  FA_HIP_CHECK(compute_units_of_current_device(&cus));
  const ExpandedPlan plan = expanded_plan(*s, cus);
  if (workspace_bytes < plan.bytes || (plan.bytes > 0 && !workspace))
    return fail(FA_ERR_SCRATCH_TOO_SMALL, "the call works in %lld bytes of workspace, %lld were given", (long long)plan.bytes,
                (long long)(workspace ? workspace_bytes : 0));

  ExpandedParams p = {};
  p.b.query_start = query_start;
  p.b.key_start = key_start;
  p.b.num_seqs = s->num_seqs;
  p.b.num_tokens = s->num_tokens;
  p.b.num_keys = s->num_keys;
  p.b.max_keys = s->max_key_len > 0 ? s->max_key_len : s->num_keys;
  p.query = reinterpret_cast<const char *>(query);
  p.key = reinterpret_cast<const char *>(key);
  p.rope_key = reinterpret_cast<const char *>(rope_key);
  p.value = reinterpret_cast<const char *>(value);
  p.out = reinterpret_cast<char *>(out);
  p.q_token_bytes = s->query_token_stride * 2;
  p.q_head_bytes = s->query_head_stride * 2;
  p.k_head_bytes = s->key_head_stride * 2;
  p.v_head_bytes = s->value_head_stride * 2;
  p.out_token_bytes = s->out_token_stride * 2;
  p.out_head_bytes = s->out_head_stride * 2;
  p.k_token_bytes = (uint32_t)(s->key_token_stride * 2);
  p.r_token_bytes = (uint32_t)(s->rope_key_token_stride * 2);
  p.v_token_bytes = (uint32_t)(s->value_token_stride * 2);
  p.score_scale_log2 = std::abs(scale) * kLog2e;
  p.query_flip = scale < 0.f ? 0x80008000u : 0u;
  p.max_query_len = s->max_query_len;
  p.num_kv_heads = s->num_heads;
  p.group = 1;
  p.window = kNoWindow;
  p.row_limit = 0;
  p.tile_groups = plan.groups;
  p.tile_o = reinterpret_cast<float *>(reinterpret_cast<char *>(workspace) + plan.tile_o);
  p.tile_ml = reinterpret_cast<float *>(reinterpret_cast<char *>(workspace) + plan.tile_ml);
  float *us = o ? o->elapsed_us : nullptr;
  KernelTimer timer(us != nullptr, o ? reinterpret_cast<hipStream_t>(o->stream) : nullptr);
  const auto of_dim = [&](auto type, auto waves) {
    using Type = decltype(type);
    constexpr int kWaves = decltype(waves)::value;
    return s->head_size == 128 ? launch_expanded_tiles<128, Type, kWaves>(p, plan, timer, us) : launch_expanded_tiles<64, Type, kWaves>(p, plan, timer, us);
  };
  const auto of_type = [&](auto waves) { return s->dtype == FA_DTYPE_BF16 ? of_dim(BF16{}, waves) : of_dim(F16{}, waves); };
  return plan.wavefronts == 8 ? of_type(std::integral_constant<int, 8>{}) : of_type(std::integral_constant<int, 4>{});
}

}  // namespace fa
