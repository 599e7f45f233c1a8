// Host launcher of ragged paged attention and differential attention (declared in include/fa_ragged.h): argument checks, which
// forms a call needs, work-group counts, workspace.
#pragma once

#include <algorithm>

#include "../../include/fa_ragged.h"
#include "launch_common.h"
#include "ragged_rows_kernel.h"
#include "ragged_tile_kernel.h"

namespace fa {

struct RaggedPlan {
  bool rows, tiles;       // which forms run
  int wavefronts;         // of a work-group of the tile form
  int tile_rows;          // rows of its tiles
  int64_t tile_bound;     // tiles per kv head, at most
  int tile_groups;        // work-groups that share all tiles; 0: a work-group for each tile
  int row_groups, row_shares;
  bool row_aligned;       // rows form: a work-group for each item, and no second kernel
  int64_t row_o, row_ml, row_seqs, tile_o, tile_ml, bytes;  // offsets into the workspace, and its size
};

inline fa_status check_ragged_shape(const fa_ragged_shape *s, int maps) {
  if (s->num_seqs < 0 || s->num_tokens < 0 || s->num_heads <= 0 || s->num_kv_heads <= 0 || s->max_blocks_per_seq <= 0 ||
      s->num_pool_blocks <= 0 || s->max_query_len <= 0 || s->max_context_len < 0)
    return fail(FA_ERR_BAD_SHAPE, "num_seqs, num_tokens and max_context_len must be >= 0; num_heads, num_kv_heads, max_blocks_per_seq, "
                                  "num_pool_blocks and max_query_len positive");
  if (s->q_dtype != FA_DTYPE_F16 && s->q_dtype != FA_DTYPE_BF16)
    return fail(FA_ERR_UNSUPPORTED_DTYPE, "q_dtype %d is neither fp16 (0) nor bf16 (1)", s->q_dtype);
  const int c = s->cache_dtype;
  if (c != FA_KV_CACHE_16BIT && c != FA_KV_CACHE_I8 && (maps == 2 || (c != FA_KV_CACHE_E5M2 && c != FA_KV_CACHE_E4M3)))
    return fail(FA_ERR_UNSUPPORTED_DTYPE, maps == 2 ? "cache_dtype %d is neither 16-bit (0) nor integers (3)"
                                                    : "cache_dtype %d is none of 16-bit (0), E5M2 (1), E4M3 (2), integers (3)", c);
  if ((s->head_size != 64 && s->head_size != 128) || s->block_size < 16 || !is_pow2(s->block_size))
    return fail(FA_ERR_UNSUPPORTED_HEAD_OR_BLOCK_SIZE,
                "Unsupported head size or block size (head_size %d must be 64 or 128, block_size %d a power of two >= 16)",
                s->head_size, s->block_size);
  if (s->num_heads % s->num_kv_heads != 0 || s->num_heads / s->num_kv_heads > kMaxGroup)
    return fail(FA_ERR_UNSUPPORTED_GROUP, "Unsupported number of queries per token: %d heads over %d kv heads (a multiple, at most %d per kv head)",
                s->num_heads, s->num_kv_heads, kMaxGroup);
  if ((int64_t)s->max_blocks_per_seq * s->block_size > 0x3fffffffLL)
    return fail(FA_ERR_BAD_SHAPE, "a block table of 2^30 tokens or more is not supported");
  // the rows form numbers 128-key units, the tile form 16-row pieces of its grid
  const int64_t keys = (int64_t)s->max_blocks_per_seq * s->block_size;
  if ((int64_t)s->num_seqs * s->num_kv_heads * (keys / kRowUnit + 2) > 0x7fffffffLL ||
      ((int64_t)s->num_tokens + s->num_seqs) * s->num_heads > 0x7fffffffLL)
    return fail(FA_ERR_BAD_SHAPE, "num_seqs x num_kv_heads x keys or num_tokens x num_heads is too large");
  // the line of tiles is as long as the sum of their keys, and cut at products with the work-groups' numbers
  if (((int64_t)s->num_tokens * s->num_heads / 32 + s->num_seqs * (int64_t)s->num_kv_heads) * (keys + 1024) > (1LL << 41))
    return fail(FA_ERR_BAD_SHAPE, "num_tokens x num_heads x keys is too large");
  return FA_OK;
}

// Which forms run, and how the work is cut; `cus`: compute units.
inline RaggedPlan ragged_plan(const fa_ragged_shape &s, int maps, int cus) {
  RaggedPlan r = {};
  const int64_t T = s.num_tokens, S = s.num_seqs, Hk = s.num_kv_heads, G = s.num_heads / s.num_kv_heads, D = s.head_size;
  if (T == 0 || S == 0) return r;
  const int64_t most = std::min<int64_t>(s.max_query_len, T);
  const int64_t table = (int64_t)s.max_blocks_per_seq * s.block_size;
  const int64_t keys = s.max_context_len > 0 ? std::min<int64_t>(s.max_context_len, table) : table;
  const bool equal = S == 1 || T == S * most;  // every sequence brings `most` tokens
  r.tiles = most * G * maps > kRowColumns;
  r.rows = G * maps <= kRowColumns && !(equal && r.tiles);
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  if (r.rows) {
    r.row_aligned = keys <= 512;
    r.row_groups = (int)std::min<int64_t>(2 * (int64_t)cus, kMaxRowGroups);
    if (!r.row_aligned) {
      r.row_shares = std::max<int>(1, r.row_groups / (int)Hk);
      const int64_t slots = (S + r.row_shares) * Hk;
      r.row_o = take(slots * kRowColumns * D * 4);
      r.row_ml = take(slots * 2 * kRowColumns * 4);
      r.row_seqs = take(S * 8);
    }
  }
  if (r.tiles) {
    // 8 wavefronts halve what K and V cost per row, and take turns in the matrix phase; 4 start and end a tile sooner, and two
    // such work-groups share a compute unit.  4 where rows do not fill more or keys are few: one prompt of 1000 tokens (8 kv heads, 4
    // query heads each, integers) 32 us with 4, 38 with 8; 16 such 225 and 226; 64 new tokens of 16 sequences of 1000 keys
    // 33 and 40; 8 prompts of 1400 tokens 191 and 182; of 1700 265 and 254; of 3000 757 and 717; 100 new tokens of 64 sequences of 2300
    // keys 370 and 343, 30 new tokens 120 and 134.  16-bit pools: 29 and 34, 219 and 214, 30 and 38, 178 and 171, 254 and 243, 714 and
    // 667, 366 and 335, 133 and 142.  Two maps, five prompts of 513 to 1546 tokens: fp16 78 and 76, bf16 88 and 87.
    r.wavefronts = most * G * maps <= 128 || keys <= 1536 ? 4 : 8;
    r.tile_rows = r.wavefronts * 32 / maps;
    const int64_t each = (most * G + r.tile_rows - 1) / r.tile_rows;
    r.tile_bound = equal ? S * each : std::min(S * each, T * G / r.tile_rows + S);
    // Tiles for each compute unit: from two on, a work-group each, longest first, keeps them all busy.  With fewer, the longest
    // tile (or two one after the other) leaves compute units idle for so many keys; shares of a line do not, but cost a second
    // kernel and their bookkeeping, about what 20 steps take: 20 new tokens of one sequence of 8000 keys 58 us as shares, 196 as
    // tiles, of 2000 keys 32 and 54, of 1000 28 and 30, of 4 sequences of 1000 keys 33 and 31, of 2000 39 and 55; 64 of 8 sequences of
    // 4000 keys 71 and 127; two prompts of 2000 tokens 110 and 95, one of 1500 58 and 45.
    const double x = (double)(r.tile_bound * Hk) / cus, mean = std::max<double>(keys - most / 2, 0);
    const bool line = x < 2 && std::max<double>(keys, x > 1 ? 2 * mean : mean) - x * mean > 20 * kTileKeys;
    if (line) {
      const int64_t resident = (int64_t)cus * (r.wavefronts == 4 ? 2 : 1);
      r.tile_groups = (int)std::max<int64_t>(8, resident / 8 * 8);  // (an eighth of the shares for each XCC)
      r.tile_o = take(2 * (int64_t)r.tile_groups * r.wavefronts * D * 32 * 4);
      r.tile_ml = take(2 * (int64_t)r.tile_groups * r.wavefronts * 128 * 4);
    }
  }
  r.bytes = at;
  return r;
}

template <int D, typename OT, int KVF, int MAPS>
inline fa_status launch_ragged_kernels(const RaggedParams &p, const RaggedPlan &plan, KernelTimer &timer, float *us) {
  const int Hk = p.num_kv_heads;
  auto timed = [&]() -> fa_status {
    if (us) FA_HIP_CHECK(timer.accumulate(0, us));
    return FA_OK;
  };
  fa_status st = FA_OK;
  if (plan.tiles) {
    const dim3 grid((unsigned)(plan.tile_groups > 0 ? plan.tile_groups : plan.tile_bound * Hk));
    const auto with_line = [&](auto ext, auto line) {
      constexpr bool kExt = decltype(ext)::value, kLine = decltype(line)::value;
      return plan.wavefronts == 8 ? timer.launch(ragged_tile_kernel<D, OT, KVF, MAPS, 8, kExt, kLine>, grid, dim3(512), 0, p)
                                  : timer.launch(ragged_tile_kernel<D, OT, KVF, MAPS, 4, kExt, kLine>, grid, dim3(256), 0, p);
    };
    const auto launch = [&](auto ext) {
      return plan.tile_groups > 0 ? with_line(ext, std::true_type{}) : with_line(ext, std::false_type{});
    };
    if constexpr (MAPS == 1) {
      FA_HIP_CHECK(p.mask_flags ? launch(std::true_type{}) : launch(std::false_type{}));
    } else {
      FA_HIP_CHECK(launch(std::false_type{}));
    }
    if ((st = timed()) != FA_OK) return st;
    if (plan.tile_groups > 1) {
      const dim3 merge((unsigned)(plan.tile_groups - 1));
      if (plan.wavefronts == 8)
        FA_HIP_CHECK(timer.launch(ragged_tile_merge_kernel<D, MAPS, 8>, merge, dim3(512), 0, p));
      else
        FA_HIP_CHECK(timer.launch(ragged_tile_merge_kernel<D, MAPS, 4>, merge, dim3(256), 0, p));
      if ((st = timed()) != FA_OK) return st;
    }
  }
  if (plan.rows) {
    const unsigned groups = plan.row_aligned ? (unsigned)(p.b.num_seqs * Hk) : (unsigned)(plan.row_shares * Hk);
    FA_HIP_CHECK(timer.launch(ragged_rows_kernel<D, OT, KVF, MAPS>, dim3(groups), dim3(256), 0, p));
    if ((st = timed()) != FA_OK || plan.row_aligned) return st;
    const int rows = std::min<int64_t>(kRowColumns / MAPS, (int64_t)p.max_query_len * p.group);
    const int64_t items = (int64_t)p.b.num_seqs * Hk;
    if (items * rows > 8 * (int64_t)plan.row_groups)  // four times what the chip holds at a time: see the second kernel
      FA_HIP_CHECK(timer.launch(ragged_rows_join_kernel<D, MAPS>, dim3((unsigned)items), dim3(512), 0, p));
    else
      FA_HIP_CHECK(timer.launch(ragged_rows_merge_kernel<D, MAPS>, dim3((unsigned)items, (unsigned)rows), dim3(512), 0, p));
    if ((st = timed()) != FA_OK) return st;
  }
  return FA_OK;
}

struct DifferentialArgs {
  const float *lambdas, *norm_weight;
  float norm_eps, out_scale;
};

inline fa_status launch_ragged_attention(void *out, const void *query, const void *key_cache, const void *value_cache,
                                         const int32_t *block_tables, const int32_t *query_start, const int32_t *context_lens,
                                         float scale, void *workspace, int64_t workspace_bytes, const fa_ragged_shape *s,
                                         const fa_paged_attention_options *o, const DifferentialArgs *diff) {
  const int maps = diff ? 2 : 1;
  fa_status st = check_ragged_shape(s, maps);
  if (st != FA_OK) return st;
  const bool nothing = s->num_tokens == 0 || s->num_seqs == 0;
  if (!nothing && (!out || !query || !key_cache || !value_cache || !block_tables || !query_start || !context_lens))
    return fail(FA_ERR_NULL_POINTER, "out, query, key_cache, value_cache, block_tables, query_start and context_lens must all be non-NULL");
  const bool kv8 = s->cache_dtype != FA_KV_CACHE_16BIT;
  const int64_t eb = kv8 ? 1 : 2;
  if (s->kv_block_stride <= 0 || s->kv_token_stride < s->head_size || s->kv_head_stride < s->head_size)
    return fail(FA_ERR_BAD_SHAPE, "kv strides must be positive and cover one head_size row");
  if ((s->kv_block_stride * eb) % 16 || (s->kv_token_stride * eb) % 16 || (s->kv_head_stride * eb) % 16)
    return fail(FA_ERR_BAD_SHAPE, "kv strides must be multiples of 16 bytes");
  if (s->kv_block_stride * eb > 0xffffffffLL || s->kv_token_stride * eb > 0xffffffffLL)
    return fail(FA_ERR_BAD_SHAPE, "kv_block_stride and kv_token_stride must be under 4 GiB");
  if (s->query_token_stride < s->head_size || s->query_head_stride < s->head_size || s->query_token_stride % 8 || s->query_head_stride % 8)
    return fail(FA_ERR_BAD_SHAPE, "query strides must cover one head_size row and be multiples of 16 bytes");
  if (((uintptr_t)out | (uintptr_t)query | (uintptr_t)key_cache | (uintptr_t)value_cache | (uintptr_t)workspace) % 16)
    return fail(FA_ERR_BAD_SHAPE, "out, query, key_cache, value_cache and workspace must be 16-byte aligned");
  if (((uintptr_t)block_tables | (uintptr_t)query_start | (uintptr_t)context_lens) % 4)
    return fail(FA_ERR_BAD_SHAPE, "block_tables, query_start and context_lens must be 4-byte aligned");
  const int flags = o ? o->mask_flags : 0;
  if (flags & ~(FA_MASK_ALIBI | FA_MASK_SOFTCAP | FA_MASK_WINDOW))
    return fail(FA_ERR_BAD_SHAPE, "mask_flags 0x%x has bits that mean nothing", flags);
  if ((flags & FA_MASK_ALIBI) && !o->alibi_slopes) return fail(FA_ERR_NULL_POINTER, "FA_MASK_ALIBI needs alibi_slopes");
  if ((flags & FA_MASK_SOFTCAP) && !(o->softcap > 0.f)) return fail(FA_ERR_BAD_SHAPE, "FA_MASK_SOFTCAP needs softcap > 0");
  if ((flags & FA_MASK_WINDOW) && o->window_left < 0) return fail(FA_ERR_BAD_SHAPE, "FA_MASK_WINDOW needs window_left >= 0");
  if (o && o->query_len > 1) return fail(FA_ERR_BAD_SHAPE, "query_len is not for ragged batches: query_start says which tokens are whose");
  if (!(scale == scale) || scale - scale != 0.f) return fail(FA_ERR_BAD_SHAPE, "scale must be finite");
  const int mode = kv8 && o ? o->kv_scale_mode : FA_KV_SCALE_TENSOR;
  if (mode != FA_KV_SCALE_TENSOR && mode != FA_KV_SCALE_HEAD && mode != FA_KV_SCALE_BLOCK)
    return fail(FA_ERR_BAD_SHAPE, "kv_scale_mode %d is none of tensor (0), head (1), block (2)", mode);
  if (mode != FA_KV_SCALE_TENSOR && (!o->k_scales || !o->v_scales))
    return fail(FA_ERR_NULL_POINTER, "kv_scale_mode %d needs k_scales and v_scales", mode);
  if (mode != FA_KV_SCALE_TENSOR && ((uintptr_t)o->k_scales | (uintptr_t)o->v_scales) % 4)
    return fail(FA_ERR_BAD_SHAPE, "k_scales and v_scales must be 4-byte aligned");
  if (s->cache_dtype == FA_KV_CACHE_I8 && mode == FA_KV_SCALE_TENSOR)
    return fail(FA_ERR_BAD_SHAPE, "pools of integers need k_scales and v_scales (kv_scale_mode head or block)");
  if (diff) {
    if (!nothing && !diff->lambdas) return fail(FA_ERR_NULL_POINTER, "lambdas must be non-NULL");
    if ((uintptr_t)diff->lambdas % 4 || (uintptr_t)diff->norm_weight % 16)
      return fail(FA_ERR_BAD_SHAPE, "lambdas must be 4-byte, norm_weight 16-byte aligned");
    if (!(diff->norm_eps >= 0.f)) return fail(FA_ERR_BAD_SHAPE, "norm_eps must be >= 0");
    if ((flags & (FA_MASK_ALIBI | FA_MASK_SOFTCAP)) || (o && o->sinks))
      return fail(FA_ERR_BAD_SHAPE, "differential attention takes a window, and neither alibi_slopes, softcap nor sinks");
  }
  if (o && o->validate_only) return FA_OK;
  if (o && o->elapsed_us) o->elapsed_us[0] = 0.f;
  if (nothing) return FA_OK;
  int cus = 0;
  FA_HIP_CHECK(compute_units_of_current_device(&cus));
  const RaggedPlan plan = ragged_plan(*s, maps, cus);
  if (workspace_bytes < plan.bytes || (plan.bytes > 0 && !workspace))
    return fail(FA_ERR_SCRATCH_TOO_SMALL, "the call works in %lld bytes of workspace, %lld were given", (long long)plan.bytes,
                (long long)(workspace ? workspace_bytes : 0));

  RaggedParams p = {};
  p.a.key_cache = reinterpret_cast<const char *>(key_cache);
  p.a.value_cache = reinterpret_cast<const char *>(value_cache);
  p.a.group = kRowColumns;
  p.a.block_shift = p.b.block_shift = ilog2(s->block_size);
  p.a.max_block_id = p.b.max_block_id = s->num_pool_blocks - 1;
  p.a.kv_block_bytes = s->kv_block_stride * eb;
  p.a.kv_token_bytes = s->kv_token_stride * eb;
  p.a.kv_head_bytes = s->kv_head_stride * eb;
  p.b.query_start = query_start;
  p.b.context_lens = context_lens;
  p.b.block_tables = block_tables;
  p.b.num_seqs = s->num_seqs;
  p.b.num_tokens = s->num_tokens;
  p.b.max_blocks_per_seq = s->max_blocks_per_seq;
  p.query = reinterpret_cast<const char *>(query);
  p.out = reinterpret_cast<char *>(out);
  p.q_token_bytes = s->query_token_stride * 2;
  p.q_head_bytes = s->query_head_stride * 2;
  p.k_scales = mode != FA_KV_SCALE_TENSOR ? o->k_scales : nullptr;
  p.v_scales = mode != FA_KV_SCALE_TENSOR ? o->v_scales : nullptr;
  p.scale_pitch = mode == FA_KV_SCALE_BLOCK ? s->num_kv_heads : 0;
  p.block_scales = mode == FA_KV_SCALE_BLOCK;
  p.tensor_scale = kv8 && mode == FA_KV_SCALE_TENSOR && o && o->fp8_scale != 0.f ? o->fp8_scale : 1.0f;
  p.sinks = o ? o->sinks : nullptr;
  p.alibi_slopes = o ? o->alibi_slopes : nullptr;
  p.softcap = o ? o->softcap : 0.f;
  p.window = (flags & FA_MASK_WINDOW) ? std::min<int32_t>(o->window_left, kNoWindow) : kNoWindow;
  p.mask_flags = flags & (FA_MASK_ALIBI | FA_MASK_SOFTCAP);
  p.score_scale_log2 = std::abs(scale) * kLog2e;
  p.query_flip = (scale < 0.f) != (p.tensor_scale < 0.f) ? 0x80008000u : 0u;
  p.q_bf16 = s->q_dtype == FA_DTYPE_BF16;
  p.num_heads = s->num_heads;
  p.num_kv_heads = s->num_kv_heads;
  p.group = s->num_heads / s->num_kv_heads;
  p.max_query_len = s->max_query_len;
  p.row_limit = plan.rows ? kRowColumns : 0;
  if (diff) {
    p.lambdas = diff->lambdas;
    p.norm_weight = diff->norm_weight;
    p.norm_eps = diff->norm_eps;
    p.out_scale = diff->out_scale;
  }
  char *space = reinterpret_cast<char *>(workspace);
  p.row_groups = plan.row_groups;
  p.row_aligned = plan.row_aligned;
  p.row_o = reinterpret_cast<float *>(space + plan.row_o);
  p.row_ml = reinterpret_cast<float *>(space + plan.row_ml);
  p.row_seqs = reinterpret_cast<int2 *>(space + plan.row_seqs);
  p.row_shares = plan.row_shares;
  p.tile_groups = plan.tile_groups;
  p.tile_o = reinterpret_cast<float *>(space + plan.tile_o);
  p.tile_ml = reinterpret_cast<float *>(space + plan.tile_ml);

  float *us = o ? o->elapsed_us : nullptr;
  KernelTimer timer(us != nullptr, o ? reinterpret_cast<hipStream_t>(o->stream) : nullptr);
  const bool d128 = s->head_size == 128;
#define FA_RAGGED(OT, KVF, MAPS)                                                       \
  (d128 ? launch_ragged_kernels<128, OT, KVF, MAPS>(p, plan, timer, us)                \
        : launch_ragged_kernels<64, OT, KVF, MAPS>(p, plan, timer, us))
  const int c = s->cache_dtype;
  if (diff) {
    if (c == FA_KV_CACHE_I8) return FA_RAGGED(F16, kKvI8, 2);
    return p.q_bf16 ? FA_RAGGED(BF16, kKv16, 2) : FA_RAGGED(F16, kKv16, 2);
  }
  if (c == FA_KV_CACHE_I8) return FA_RAGGED(F16, kKvI8, 1);
  if (c == FA_KV_CACHE_E4M3) return FA_RAGGED(F16, kKvE4M3, 1);
  if (c == FA_KV_CACHE_E5M2) return FA_RAGGED(F16, kKvE5M2, 1);
  return p.q_bf16 ? FA_RAGGED(BF16, kKv16, 1) : FA_RAGGED(F16, kKv16, 1);
#undef FA_RAGGED
}

}  // namespace fa
