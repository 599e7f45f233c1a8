// extern "C" surface of libfa_paged_attention.so for ragged batches (include/fa_ragged.h): append, attention, differential attention.
#include "launch_kv_cache_append.h"
#include "launch_ragged_attention.h"

#define FA_EXPORT extern "C" __attribute__((visibility("default")))

namespace {

// shape and options as the library works with them
template <typename Shape>
fa_status read_ragged(const Shape *shape, size_t least, const fa_paged_attention_options *options, Shape *sh, fa::CallStructs *c) {
  fa::error_buffer()[0] = 0;
  if (!shape) return fa::fail(FA_ERR_NULL_POINTER, "shape is NULL");
  const fa_status st = fa::read_versioned(shape, sh, least, "shape");
  return st == FA_OK ? fa::read_options(options, c) : st;
}
constexpr size_t kAppendLeast = offsetof(fa_kv_cache_append_shape, fp8_scale) + sizeof(float);
constexpr size_t kRaggedLeast = offsetof(fa_ragged_shape, max_context_len) + sizeof(int32_t);

}  // namespace

FA_EXPORT int32_t fa_kv_cache_append(const void *query, void *query_out, const void *key, const void *value, void *key_cache,
                                     void *value_cache, const float *cos_sin, const int32_t *block_tables,
                                     const int32_t *query_start, const int32_t *context_lens, float *k_scales, float *v_scales,
                                     const fa_kv_cache_append_shape *shape, const fa_paged_attention_options *options) {
  fa_kv_cache_append_shape sh;
  fa::CallStructs c;
  const fa_status st = read_ragged(shape, kAppendLeast, options, &sh, &c);
  if (st != FA_OK) return st;
  return fa::launch_kv_cache_append(query, query_out, key, value, key_cache, value_cache, cos_sin, block_tables, query_start,
                                    context_lens, k_scales, v_scales, &sh, c.options());
}

FA_EXPORT int64_t fa_paged_attention_ragged_workspace_bytes(const fa_ragged_shape *shape, int32_t maps) {
  fa_ragged_shape sh;
  fa::CallStructs c;
  if (read_ragged(shape, kRaggedLeast, nullptr, &sh, &c) != FA_OK || (maps != 1 && maps != 2) || fa::check_ragged_shape(&sh, maps) != FA_OK)
    return 0;
  int cus = 0;
  if (fa::compute_units_of_current_device(&cus) != hipSuccess) return 0;
  return fa::ragged_plan(sh, maps, cus).bytes;
}

FA_EXPORT int32_t fa_paged_attention_ragged(void *out, const void *query, const void *key_cache, const void *value_cache,
                                            const int32_t *block_tables, const int32_t *query_start, const int32_t *context_lens,
                                            float scale, void *workspace, int64_t workspace_bytes, const fa_ragged_shape *shape,
                                            const fa_paged_attention_options *options) {
  fa_ragged_shape sh;
  fa::CallStructs c;
  const fa_status st = read_ragged(shape, kRaggedLeast, options, &sh, &c);
  if (st != FA_OK) return st;
  return fa::launch_ragged_attention(out, query, key_cache, value_cache, block_tables, query_start, context_lens, scale, workspace,
                                     workspace_bytes, &sh, c.options(), nullptr);
}

FA_EXPORT int32_t fa_paged_attention_differential(void *out, const void *query, const void *key_cache, const void *value_cache,
                                                  const int32_t *block_tables, const int32_t *query_start,
                                                  const int32_t *context_lens, float scale, const float *lambdas,
                                                  const float *norm_weight, float norm_eps, float out_scale, void *workspace,
                                                  int64_t workspace_bytes, const fa_ragged_shape *shape,
                                                  const fa_paged_attention_options *options) {
  fa_ragged_shape sh;
  fa::CallStructs c;
  const fa_status st = read_ragged(shape, kRaggedLeast, options, &sh, &c);
  if (st != FA_OK) return st;
  const fa::DifferentialArgs diff = {lambdas, norm_weight, norm_eps, out_scale};
  return fa::launch_ragged_attention(out, query, key_cache, value_cache, block_tables, query_start, context_lens, scale, workspace,
                                     workspace_bytes, &sh, c.options(), &diff);
}
