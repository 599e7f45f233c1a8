// extern "C" surface of libfa_paged_attention.so for latent attention (include/fa_latent.h): append, read-back, absorbed and expanded
// attention.
#include "launch_latent.h"

#define FA_EXPORT extern "C" __attribute__((visibility("default")))

namespace {

// shape and options as the library works with them
template <typename Shape>
fa_status read_latent(const Shape *shape, const fa_paged_attention_options *options, Shape *sh, fa::CallStructs *c) {
  fa::error_buffer()[0] = 0;
  if (!shape) return fa::fail(FA_ERR_NULL_POINTER, "shape is NULL");
  const fa_status st = fa::read_versioned(shape, sh, sizeof(Shape), "shape");  // every field of the first revision is needed
  return st == FA_OK ? fa::read_options(options, c) : st;
}

}  // namespace

FA_EXPORT int32_t fa_latent_cache_append(const void *latent, const void *rope_key, void *cache, const float *norm_weight, const float *cos_sin,
                                         const void *query_rope, void *query_rope_out, float *scales, const int32_t *block_tables,
                                         const int32_t *query_start, const int32_t *context_lens, const fa_latent_append_shape *shape,
                                         const fa_paged_attention_options *options) {
  fa_latent_append_shape sh;
  fa::CallStructs c;
  const fa_status st = read_latent(shape, options, &sh, &c);
  if (st != FA_OK) return st;
  return fa::launch_latent_cache_append(latent, rope_key, cache, norm_weight, cos_sin, query_rope, query_rope_out, scales, block_tables,
                                        query_start, context_lens, &sh, c.options());
}

FA_EXPORT int32_t fa_latent_cache_gather(void *out, const void *cache, const float *scales, const int32_t *block_tables, const int32_t *row_start,
                                         const int32_t *first_keys, const fa_latent_gather_shape *shape, const fa_paged_attention_options *options) {
  fa_latent_gather_shape sh;
  fa::CallStructs c;
  const fa_status st = read_latent(shape, options, &sh, &c);
  if (st != FA_OK) return st;
  return fa::launch_latent_cache_gather(out, cache, scales, block_tables, row_start, first_keys, &sh, c.options());
}

FA_EXPORT int64_t fa_paged_attention_latent_workspace_bytes(const fa_latent_attention_shape *shape) {
  fa_latent_attention_shape sh;
  fa::CallStructs c;
  int cus = 0;
  if (read_latent(shape, nullptr, &sh, &c) != FA_OK || fa::check_latent_attention_shape(&sh) != FA_OK ||
      fa::compute_units_of_current_device(&cus) != hipSuccess)
    return 0;
  return fa::latent_plan(sh, cus).bytes;
}

FA_EXPORT int32_t fa_paged_attention_latent(void *out, const void *query_latent, const void *query_rope, const void *cache, const float *scales,
                                            const int32_t *block_tables, const int32_t *query_start, const int32_t *context_lens, float scale,
                                            void *workspace, int64_t workspace_bytes, const fa_latent_attention_shape *shape,
                                            const fa_paged_attention_options *options) {
  fa_latent_attention_shape sh;
  fa::CallStructs c;
  const fa_status st = read_latent(shape, options, &sh, &c);
  if (st != FA_OK) return st;
  return fa::launch_latent_attention(out, query_latent, query_rope, cache, scales, block_tables, query_start, context_lens, scale, workspace,
                                     workspace_bytes, &sh, c.options());
}

FA_EXPORT int64_t fa_attention_latent_expanded_workspace_bytes(const fa_latent_expanded_shape *shape) {
  fa_latent_expanded_shape sh;
  fa::CallStructs c;
  int cus = 0;
  if (read_latent(shape, nullptr, &sh, &c) != FA_OK || fa::check_latent_expanded_shape(&sh) != FA_OK ||
      fa::compute_units_of_current_device(&cus) != hipSuccess)
    return 0;
  return fa::expanded_plan(sh, cus).bytes;
}

FA_EXPORT int32_t fa_attention_latent_expanded(void *out, const void *query, const void *key, const void *rope_key, const void *value,
                                               const int32_t *query_start, const int32_t *key_start, float scale, void *workspace,
                                               int64_t workspace_bytes, const fa_latent_expanded_shape *shape,
                                               const fa_paged_attention_options *options) {
  fa_latent_expanded_shape sh;
  fa::CallStructs c;
  const fa_status st = read_latent(shape, options, &sh, &c);
  if (st != FA_OK) return st;
  return fa::launch_latent_expanded(out, query, key, rope_key, value, query_start, key_start, scale, workspace, workspace_bytes, &sh, c.options());
}
