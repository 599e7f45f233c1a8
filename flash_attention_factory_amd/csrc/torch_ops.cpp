// torch.ops.fa_amd in native code: from the dispatcher to the C ABI without Python.
//
// A decode step issues these operators by the dozen, most of them for kernels of 5 to 30 us, and a call through
// torch.library.custom_op and ctypes costs the host 24 us (10 of them in three Python kernels of the dispatcher,
// 14 in the argument checks and the ctypes call).  Through this file it costs 5 to 6: an append and an attention of four
// short sequences 44 -> 11 us, calls whose kernels take less than the host did 25 to 28 -> 17 to 19 us.
//
// The operators that torch_ops.py defines in Python (namespace fa_amd_py, the same schemas) stay what says which
// calls are valid and what an invalid one raises.  A native kernel makes the same checks, launches what passes
// them, and hands every other call -- a failed check, a status that is not FA_OK, scratch that needs a warning,
// an input that requires grad -- to the Python operator, which raises or does what it always did.
#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <atomic>
#include <limits>

#include "../../include/fa_kv_cache.h"
#include "../../include/fa_latent.h"
#include "../../include/fa_paged_attention.h"
#include "../../include/fa_ragged.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

// The C ABI's entry points, as the process has loaded them (fa_torch_ops_bind); null until then.
struct Entries {
  decltype(&fa_paged_attention_loop) loop, fp8_loop;
  decltype(&fa_paged_attention_reduce) reduce, fp8_reduce;
  decltype(&fa_kv_cache_write) kv_cache_write;
  decltype(&fa_paged_attention_loop_workspace_bytes) workspace_bytes;
  decltype(&fa_kv_cache_append) kv_cache_append;
  decltype(&fa_paged_attention_ragged) ragged;
  decltype(&fa_paged_attention_differential) differential;
  decltype(&fa_paged_attention_ragged_workspace_bytes) ragged_workspace_bytes;
  decltype(&fa_latent_cache_append) latent_append;
  decltype(&fa_latent_cache_gather) latent_gather;
  decltype(&fa_paged_attention_latent) latent;
  decltype(&fa_paged_attention_latent_workspace_bytes) latent_workspace_bytes;
  decltype(&fa_attention_latent_expanded) latent_expanded;
  decltype(&fa_attention_latent_expanded_workspace_bytes) latent_expanded_workspace_bytes;
};
Entries entries = {};

// The Python operators have given their one warning of scratch that a wide table could outgrow
// (fa_torch_ops_capacity_warned): from then on such a call has nothing to say and is launched here.
std::atomic<bool> capacity_warned{false};

bool fits_int32(int64_t v) { return v >= std::numeric_limits<int32_t>::min() && v <= std::numeric_limits<int32_t>::max(); }

bool is_16bit(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16; }
bool is_byte_cache(at::ScalarType t) { return t == at::kFloat8_e5m2 || t == at::kFloat8_e4m3fn || t == at::kByte; }

// Block ids, heads and rows are checked against key_cache alone, so value_cache has to hold at least as much.
bool covers(const Tensor &value_cache, const Tensor &key_cache) {
  for (int64_t d = 0; d < key_cache.dim(); ++d)
    if (value_cache.size(d) < key_cache.size(d)) return false;
  return true;
}

bool same_device(const Tensor &anchor, const Tensor &t) { return t.device() == anchor.device(); }
bool same_device(const Tensor &anchor, const OptTensor &t) { return !t.has_value() || t->device() == anchor.device(); }

// k_scales / v_scales into the options; false: not a pair the kernels take.
bool set_scales(fa_paged_attention_options &op, const OptTensor &k_scales, const OptTensor &v_scales, int64_t kv_heads,
                int64_t blocks, const Tensor &anchor) {
  if (!k_scales.has_value() && !v_scales.has_value()) return true;
  if (!k_scales.has_value() || !v_scales.has_value()) return false;
  for (const Tensor *t : {&*k_scales, &*v_scales})
    if (t->scalar_type() != at::kFloat || !t->is_contiguous() || !same_device(anchor, *t) || t->sizes() != k_scales->sizes())
      return false;
  if (k_scales->dim() == 1 && k_scales->size(0) == kv_heads) op.kv_scale_mode = FA_KV_SCALE_HEAD;
  else if (k_scales->dim() == 2 && k_scales->size(0) == blocks && k_scales->size(1) == kv_heads) op.kv_scale_mode = FA_KV_SCALE_BLOCK;
  else return false;
  op.k_scales = static_cast<const float *>(k_scales->const_data_ptr());
  op.v_scales = static_cast<const float *>(v_scales->const_data_ptr());
  return true;
}

struct Scratch { const Tensor &exp_sums, &max_logits, &tmp_out; };

// One attention call; false: the Python operator has to see it.
bool attend(const Tensor &out, const Scratch *scratch, const Tensor &query, const Tensor &key_cache, const Tensor &value_cache,
            const Tensor &block_tables, const Tensor &context_lens, double scale, bool fp8, double fp8_scale,
            int64_t partition_size, const OptTensor &sinks, const OptTensor &alibi_slopes, double softcap, int64_t window_left,
            const OptTensor &k_scales, const OptTensor &v_scales, int64_t max_context_len) {
  if (!entries.loop || !query.is_cuda()) return false;
  for (const Tensor *t : {&out, &key_cache, &value_cache, &block_tables, &context_lens})
    if (!same_device(query, *t)) return false;
  if (!same_device(query, sinks) || !same_device(query, alibi_slopes)) return false;
  if (!query.is_contiguous() || !out.is_contiguous() || !block_tables.is_contiguous() || !context_lens.is_contiguous()) return false;
  const auto q_type = query.scalar_type(), kv_type = key_cache.scalar_type();
  if (!is_16bit(q_type) || out.scalar_type() != q_type) return false;
  if (block_tables.scalar_type() != at::kInt || context_lens.scalar_type() != at::kInt) return false;
  if ((fp8 ? !is_byte_cache(kv_type) : kv_type != q_type) || value_cache.scalar_type() != kv_type) return false;
  if (key_cache.dim() != 4 || key_cache.stride(3) != 1 || value_cache.strides() != key_cache.strides()) return false;
  if (!covers(value_cache, key_cache)) return false;
  if ((query.dim() != 3 && query.dim() != 4) || out.sizes() != query.sizes()) return false;
  const int64_t S = query.size(0), QL = query.dim() == 4 ? query.size(1) : 1, H = query.size(-2), D = query.size(-1);
  const int64_t blocks = key_cache.size(0), block_size = key_cache.size(1), kv_heads = key_cache.size(2);
  if (block_tables.dim() != 2 || block_tables.size(0) != S || context_lens.numel() != S || key_cache.size(3) != D) return false;
  if (kv_heads <= 0 || H % kv_heads != 0) return false;
  for (int64_t v : {S, QL, H, D, blocks, block_size, kv_heads, block_tables.size(1), partition_size, window_left, max_context_len})
    if (!fits_int32(v)) return false;
  if (sinks.has_value() && (sinks->scalar_type() != q_type || sinks->numel() != H || !sinks->is_contiguous())) return false;

  fa_paged_attention_shape sh = FA_PAGED_ATTENTION_SHAPE_INIT;
  sh.num_seqs = (int32_t)S;
  sh.num_heads = (int32_t)H;
  sh.num_kv_heads = (int32_t)kv_heads;
  sh.head_size = (int32_t)D;
  sh.block_size = (int32_t)block_size;
  sh.max_blocks_per_seq = (int32_t)block_tables.size(1);
  sh.max_num_partitions = 1;
  sh.partition_size = (int32_t)partition_size;
  sh.kv_block_stride = key_cache.stride(0);
  sh.kv_token_stride = key_cache.stride(1);
  sh.kv_head_stride = key_cache.stride(2);
  sh.num_pool_blocks = (int32_t)blocks;
  sh.q_dtype = q_type == at::kBFloat16 ? FA_DTYPE_BF16 : FA_DTYPE_F16;

  fa_paged_attention_options_workspace full = FA_PAGED_ATTENTION_OPTIONS_WORKSPACE_INIT;
  fa_paged_attention_options &op = full.options;
  op.sinks = sinks.has_value() ? sinks->const_data_ptr() : nullptr;
  op.softcap = (float)softcap;
  op.fp8_scale = (float)fp8_scale;
  if (alibi_slopes.has_value()) {
    if (alibi_slopes->scalar_type() != at::kFloat || !alibi_slopes->is_contiguous() || alibi_slopes->numel() != H) return false;
    op.alibi_slopes = static_cast<const float *>(alibi_slopes->const_data_ptr());
    op.mask_flags |= FA_MASK_ALIBI;
  }
  if (softcap > 0.0) op.mask_flags |= FA_MASK_SOFTCAP;
  if (window_left >= 0) {
    op.mask_flags |= FA_MASK_WINDOW;
    op.window_left = (int32_t)window_left;
  }
  op.query_len = (int32_t)QL;
  if (!fp8 && (k_scales.has_value() || v_scales.has_value())) return false;
  if (!set_scales(op, k_scales, v_scales, kv_heads, blocks, query)) return false;
  op.kv_fp8_format = kv_type == at::kFloat8_e4m3fn ? FA_FP8_E4M3 : FA_FP8_E5M2;

  if (scratch) {
    for (const Tensor *t : {&scratch->exp_sums, &scratch->max_logits, &scratch->tmp_out})
      if (!same_device(query, *t) || t->scalar_type() != at::kFloat || !t->is_contiguous() || t->dim() < 1) return false;
    const int64_t partitions = scratch->max_logits.size(-1);
    const int64_t slots = S * QL * H * partitions;
    if (!fits_int32(partitions) || scratch->max_logits.numel() != slots || scratch->exp_sums.numel() != slots ||
        scratch->tmp_out.numel() != slots * D)
      return false;
    sh.max_num_partitions = (int32_t)partitions;
    if (max_context_len < 0) {  // unknown: the Python operator warns, once, where the scratch arrays may be too small
      const int64_t size = partition_size > 0 ? partition_size : (D == 64 ? 256 : 512);
      if (scratch->exp_sums.size(-1) * size < block_tables.size(1) * block_size && !capacity_warned.load(std::memory_order_relaxed))
        return false;
      max_context_len = 0;
    }
  }

  const c10::DeviceGuard guard(query.device());
  op.stream = c10::hip::getCurrentHIPStream(query.device().index()).stream();
  const auto *tables = static_cast<const int32_t *>(block_tables.const_data_ptr());
  const auto *lens = static_cast<const int32_t *>(context_lens.const_data_ptr());
  void *o = out.data_ptr();
  const void *q = query.const_data_ptr(), *k = key_cache.const_data_ptr(), *v = value_cache.const_data_ptr();
  if (scratch)
    return (fp8 ? entries.fp8_reduce : entries.reduce)(
               o, q, k, v, tables, lens, (float)scale, (int32_t)max_context_len, static_cast<float *>(scratch->exp_sums.data_ptr()),
               static_cast<float *>(scratch->max_logits.data_ptr()), static_cast<float *>(scratch->tmp_out.data_ptr()), &sh,
               &op) == FA_OK;
  Tensor space;
  if (const int64_t need = entries.workspace_bytes(&sh, &op, fp8); need > 0) {  // see fa_paged_attention_options_workspace
    try {
      space = at::empty({need}, query.options().dtype(at::kByte));
      full.workspace = space.data_ptr();
      full.workspace_bytes = need;
    } catch (const c10::OutOfMemoryError &) {  // the call needs none
    }
  }
  return (fp8 ? entries.fp8_loop : entries.loop)(o, q, k, v, tables, lens, (float)scale, 0, &sh, &op) == FA_OK;
}

bool append(const Tensor &key, const Tensor &value, const Tensor &key_cache, const Tensor &value_cache, const Tensor &slot_mapping,
            double fp8_scale, const OptTensor &k_scales, const OptTensor &v_scales) {
  if (!entries.loop || !key.is_cuda()) return false;
  for (const Tensor *t : {&value, &key_cache, &value_cache, &slot_mapping})
    if (!same_device(key, *t)) return false;
  const auto type = key.scalar_type(), kv_type = key_cache.scalar_type();
  if (!is_16bit(type) || value.scalar_type() != type) return false;
  if (key.dim() != 3 || key.stride(2) != 1 || value.sizes() != key.sizes() || value.strides() != key.strides()) return false;
  const bool fp8 = is_byte_cache(kv_type);
  if ((!fp8 && kv_type != type) || value_cache.scalar_type() != kv_type) return false;
  if (key_cache.dim() != 4 || key_cache.stride(3) != 1 || value_cache.strides() != key_cache.strides() ||
      !covers(value_cache, key_cache) || key_cache.size(2) != key.size(1) || key_cache.size(3) != key.size(2))
    return false;
  if (slot_mapping.scalar_type() != at::kLong || !slot_mapping.is_contiguous() || slot_mapping.numel() != key.size(0)) return false;
  for (int64_t v : {key.size(0), key.size(1), key.size(2), key_cache.size(1)})
    if (!fits_int32(v)) return false;
  fa_kv_cache_write_shape sh = FA_KV_CACHE_WRITE_SHAPE_INIT;
  sh.num_tokens = (int32_t)key.size(0);
  sh.num_kv_heads = (int32_t)key.size(1);
  sh.head_size = (int32_t)key.size(2);
  sh.block_size = (int32_t)key_cache.size(1);
  sh.kv_block_stride = key_cache.stride(0);
  sh.kv_token_stride = key_cache.stride(1);
  sh.kv_head_stride = key_cache.stride(2);
  sh.src_token_stride = key.stride(0);
  sh.src_head_stride = key.stride(1);
  sh.src_dtype = type == at::kBFloat16 ? FA_DTYPE_BF16 : FA_DTYPE_F16;
  sh.cache_dtype = !fp8 ? FA_KV_CACHE_16BIT : kv_type == at::kFloat8_e4m3fn ? FA_KV_CACHE_E4M3 : FA_KV_CACHE_E5M2;
  sh.num_pool_blocks = key_cache.size(0);
  fa_paged_attention_options op = FA_PAGED_ATTENTION_OPTIONS_INIT;
  op.fp8_scale = (float)fp8_scale;
  if (!fp8 && (k_scales.has_value() || v_scales.has_value())) return false;
  if (!set_scales(op, k_scales, v_scales, key.size(1), key_cache.size(0), key)) return false;
  const c10::DeviceGuard guard(key.device());
  op.stream = c10::hip::getCurrentHIPStream(key.device().index()).stream();
  return entries.kv_cache_write(key.const_data_ptr(), value.const_data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(),
                                static_cast<const int64_t *>(slot_mapping.const_data_ptr()), &sh, &op) == FA_OK;
}

// ---- ragged batches ----

const float *floats(const OptTensor &t) { return t.has_value() ? static_cast<const float *>(t->const_data_ptr()) : nullptr; }
bool is_floats(const Tensor &t) { return t.scalar_type() == at::kFloat && t.is_contiguous(); }
const int32_t *ints(const Tensor &t) { return static_cast<const int32_t *>(t.const_data_ptr()); }

// The fa_kv_cache_dtype of a pair of pools for rows of `type`; -1: not a pair the kernels take.
int32_t cache_dtype(const Tensor &key_cache, const Tensor &value_cache, at::ScalarType type) {
  const auto kv = key_cache.scalar_type();
  if (value_cache.scalar_type() != kv) return -1;
  if (kv == type) return FA_KV_CACHE_16BIT;
  if (kv == at::kChar) return FA_KV_CACHE_I8;
  return kv == at::kFloat8_e4m3fn ? FA_KV_CACHE_E4M3 : is_byte_cache(kv) ? FA_KV_CACHE_E5M2 : -1;
}

// Sequences of a batch, its arrays checked; -1: not arrays the kernels take.
int64_t batch_of(const Tensor &block_tables, const Tensor &query_start, const Tensor &context_lens) {
  for (const Tensor *t : {&block_tables, &query_start, &context_lens})
    if (t->scalar_type() != at::kInt || !t->is_contiguous()) return -1;
  const int64_t S = context_lens.numel();
  if (context_lens.dim() != 1 || block_tables.dim() != 2 || block_tables.size(0) != S || query_start.dim() != 1 ||
      query_start.numel() != S + 1 || !fits_int32(S) || !fits_int32(block_tables.size(1)))
    return -1;
  return S;
}

bool pools_fit(const Tensor &key_cache, const Tensor &value_cache, int64_t head_size) {
  if (key_cache.dim() != 4 || key_cache.stride(3) != 1 || value_cache.strides() != key_cache.strides() || !covers(value_cache, key_cache) ||
      key_cache.size(3) != head_size)
    return false;
  for (int64_t d = 0; d < 4; ++d)
    if (!fits_int32(key_cache.size(d))) return false;
  return true;
}

// fa_kv_scale of a pair of scale tensors; -1: not a pair the kernels take.
int32_t scale_mode(const OptTensor &k_scales, const OptTensor &v_scales, const Tensor &key_cache) {
  if (k_scales.has_value() != v_scales.has_value()) return -1;
  if (!k_scales.has_value()) return FA_KV_SCALE_TENSOR;
  if (!is_floats(*k_scales) || !is_floats(*v_scales) || k_scales->sizes() != v_scales->sizes()) return -1;
  const int64_t heads = key_cache.size(2);
  if (k_scales->dim() == 1 && k_scales->size(0) == heads) return FA_KV_SCALE_HEAD;
  if (k_scales->dim() == 2 && k_scales->size(0) == key_cache.size(0) && k_scales->size(1) == heads) return FA_KV_SCALE_BLOCK;
  return -1;
}

bool ragged_append(const Tensor &key, const Tensor &value, const Tensor &key_cache, const Tensor &value_cache,
                   const Tensor &block_tables, const Tensor &query_start, const Tensor &context_lens, const OptTensor &cos_sin,
                   const OptTensor &query, const OptTensor &query_out, const OptTensor &k_scales, const OptTensor &v_scales,
                   double fp8_scale, bool interleaved) {
  if (!entries.loop || !key.is_cuda()) return false;
  for (const Tensor *t : {&value, &key_cache, &value_cache, &block_tables, &query_start, &context_lens})
    if (!same_device(key, *t)) return false;
  for (const OptTensor *t : {&cos_sin, &query, &query_out, &k_scales, &v_scales})
    if (!same_device(key, *t)) return false;
  const auto type = key.scalar_type();
  if (!is_16bit(type) || query.has_value() != query_out.has_value()) return false;
  auto rows = [&](const Tensor &t) {
    return t.scalar_type() == type && t.dim() == 3 && t.stride(2) == 1 && t.size(0) == key.size(0) && t.size(2) == key.size(2) &&
           fits_int32(t.size(0)) && fits_int32(t.size(1)) && fits_int32(t.size(2));
  };
  if (!rows(key) || !rows(value) || value.size(1) != key.size(1)) return false;
  if (query.has_value() && (!rows(*query) || !rows(*query_out) || query->size(1) != query_out->size(1))) return false;
  if (!pools_fit(key_cache, value_cache, key.size(2)) || key_cache.size(2) != key.size(1)) return false;
  const int64_t S = batch_of(block_tables, query_start, context_lens);
  const int32_t cache = cache_dtype(key_cache, value_cache, type), mode = scale_mode(k_scales, v_scales, key_cache);
  if (S < 0 || cache < 0 || mode < 0 || (cache == FA_KV_CACHE_16BIT && k_scales.has_value())) return false;
  fa_kv_cache_append_shape sh = FA_KV_CACHE_APPEND_SHAPE_INIT;
  sh.num_seqs = (int32_t)S;
  sh.num_tokens = (int32_t)key.size(0);
  sh.num_kv_heads = (int32_t)key.size(1);
  sh.head_size = (int32_t)key.size(2);
  sh.block_size = (int32_t)key_cache.size(1);
  sh.max_blocks_per_seq = (int32_t)block_tables.size(1);
  sh.kv_block_stride = key_cache.stride(0);
  sh.kv_token_stride = key_cache.stride(1);
  sh.kv_head_stride = key_cache.stride(2);
  sh.key_token_stride = key.stride(0);
  sh.key_head_stride = key.stride(1);
  sh.value_token_stride = value.stride(0);
  sh.value_head_stride = value.stride(1);
  if (query.has_value()) {
    sh.num_heads = (int32_t)query->size(1);
    sh.query_token_stride = query->stride(0);
    sh.query_head_stride = query->stride(1);
    sh.query_out_token_stride = query_out->stride(0);
    sh.query_out_head_stride = query_out->stride(1);
  }
  if (cos_sin.has_value()) {
    if (!is_floats(*cos_sin) || cos_sin->dim() != 2 || cos_sin->numel() == 0 || !fits_int32(cos_sin->size(0)) || !fits_int32(cos_sin->size(1)))
      return false;
    sh.max_positions = (int32_t)cos_sin->size(0);
    sh.rotary_dim = (int32_t)cos_sin->size(1);
  }
  sh.src_dtype = type == at::kBFloat16 ? FA_DTYPE_BF16 : FA_DTYPE_F16;
  sh.cache_dtype = cache;
  sh.kv_scale_mode = mode;
  sh.num_pool_blocks = (int32_t)key_cache.size(0);
  sh.interleaved = interleaved;
  sh.fp8_scale = (float)fp8_scale;
  fa_paged_attention_options op = FA_PAGED_ATTENTION_OPTIONS_INIT;
  const c10::DeviceGuard guard(key.device());
  op.stream = c10::hip::getCurrentHIPStream(key.device().index()).stream();
  return entries.kv_cache_append(query.has_value() ? query->const_data_ptr() : nullptr, query_out.has_value() ? query_out->data_ptr() : nullptr,
                                 key.const_data_ptr(), value.const_data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(),
                                 floats(cos_sin), ints(block_tables), ints(query_start), ints(context_lens),
                                 const_cast<float *>(floats(k_scales)), const_cast<float *>(floats(v_scales)), &sh, &op) == FA_OK;
}

struct Differential {
  const Tensor &lambdas;
  const OptTensor &norm_weight;
  double norm_eps, out_scale;
};

bool ragged_attend(const Tensor &out, const Tensor &query, const Tensor &key_cache, const Tensor &value_cache,
                   const Tensor &block_tables, const Tensor &query_start, const Tensor &context_lens, double scale,
                   int64_t max_query_len, int64_t max_context_len, double fp8_scale, const OptTensor &k_scales,
                   const OptTensor &v_scales, const OptTensor &sinks, const OptTensor &alibi_slopes, double softcap,
                   int64_t window_left, const Differential *diff) {
  if (!entries.loop || !query.is_cuda()) return false;
  for (const Tensor *t : {&out, &key_cache, &value_cache, &block_tables, &query_start, &context_lens})
    if (!same_device(query, *t)) return false;
  for (const OptTensor *t : {&k_scales, &v_scales, &sinks, &alibi_slopes})
    if (!same_device(query, *t)) return false;
  const auto type = query.scalar_type();
  if (!is_16bit(type) || query.dim() != 3 || (query.size(2) > 1 && query.stride(2) != 1)) return false;
  if (out.scalar_type() != type || out.sizes() != query.sizes() || !out.is_contiguous()) return false;
  if (!pools_fit(key_cache, value_cache, query.size(2))) return false;
  const int64_t S = batch_of(block_tables, query_start, context_lens), H = query.size(1);
  const int32_t cache = cache_dtype(key_cache, value_cache, type), mode = scale_mode(k_scales, v_scales, key_cache);
  if (S < 0 || cache < 0 || mode < 0 || (cache == FA_KV_CACHE_16BIT && k_scales.has_value())) return false;
  for (int64_t v : {query.size(0), H, query.size(2), max_query_len, max_context_len, window_left})
    if (!fits_int32(v)) return false;
  fa_ragged_shape sh = FA_RAGGED_SHAPE_INIT;
  sh.num_seqs = (int32_t)S;
  sh.num_tokens = (int32_t)query.size(0);
  sh.num_heads = (int32_t)H;
  sh.num_kv_heads = (int32_t)key_cache.size(2);
  sh.head_size = (int32_t)query.size(2);
  sh.block_size = (int32_t)key_cache.size(1);
  sh.max_blocks_per_seq = (int32_t)block_tables.size(1);
  sh.kv_block_stride = key_cache.stride(0);
  sh.kv_token_stride = key_cache.stride(1);
  sh.kv_head_stride = key_cache.stride(2);
  sh.query_token_stride = query.stride(0);
  sh.query_head_stride = query.stride(1);
  sh.q_dtype = type == at::kBFloat16 ? FA_DTYPE_BF16 : FA_DTYPE_F16;
  sh.cache_dtype = cache;
  sh.num_pool_blocks = (int32_t)key_cache.size(0);
  sh.max_query_len = (int32_t)max_query_len;
  sh.max_context_len = (int32_t)max_context_len;
  fa_paged_attention_options op = FA_PAGED_ATTENTION_OPTIONS_INIT;
  if (sinks.has_value()) {
    if (sinks->scalar_type() != type || sinks->numel() != H || !sinks->is_contiguous()) return false;
    op.sinks = sinks->const_data_ptr();
  }
  if (alibi_slopes.has_value()) {
    if (!is_floats(*alibi_slopes) || alibi_slopes->numel() != H) return false;
    op.alibi_slopes = floats(alibi_slopes);
    op.mask_flags |= FA_MASK_ALIBI;
  }
  if (softcap > 0.0) {
    op.mask_flags |= FA_MASK_SOFTCAP;
    op.softcap = (float)softcap;
  }
  if (window_left >= 0) {
    op.mask_flags |= FA_MASK_WINDOW;
    op.window_left = (int32_t)window_left;
  }
  op.fp8_scale = (float)fp8_scale;
  op.kv_scale_mode = mode;
  op.k_scales = floats(k_scales);
  op.v_scales = floats(v_scales);
  if (diff) {
    if (!same_device(query, diff->lambdas) || !same_device(query, diff->norm_weight)) return false;
    if (!is_floats(diff->lambdas) || diff->lambdas.numel() != H) return false;
    if (diff->norm_weight.has_value() && (!is_floats(*diff->norm_weight) || diff->norm_weight->numel() != query.size(2))) return false;
  }
  const c10::DeviceGuard guard(query.device());
  op.stream = c10::hip::getCurrentHIPStream(query.device().index()).stream();
  const int64_t need = entries.ragged_workspace_bytes(&sh, diff ? 2 : 1);
  Tensor space;
  void *at_space = nullptr;
  if (need > 0) {
    space = at::empty({need}, query.options().dtype(at::kByte));
    at_space = space.data_ptr();
  }
  if (diff)
    return entries.differential(out.data_ptr(), query.const_data_ptr(), key_cache.const_data_ptr(), value_cache.const_data_ptr(),
                                ints(block_tables), ints(query_start), ints(context_lens), (float)scale,
                                static_cast<const float *>(diff->lambdas.const_data_ptr()), floats(diff->norm_weight),
                                (float)diff->norm_eps, (float)diff->out_scale, at_space, need, &sh, &op) == FA_OK;
  return entries.ragged(out.data_ptr(), query.const_data_ptr(), key_cache.const_data_ptr(), value_cache.const_data_ptr(),
                        ints(block_tables), ints(query_start), ints(context_lens), (float)scale, at_space, need, &sh, &op) == FA_OK;
}

// ---- latent attention ---------------------------------------------------------------------------

constexpr int64_t kRope = 64;  // elements of a latent pool's rotated part

// The fa_kv_cache_dtype of a latent pool for rows of `type`; -1: not a pool the kernels take.
int32_t latent_pool(const Tensor &cache, const OptTensor &scales, at::ScalarType type) {
  if (cache.dim() != 3 || cache.stride(2) != 1 || cache.size(2) <= kRope) return -1;
  for (int64_t d = 0; d < 3; ++d)
    if (!fits_int32(cache.size(d))) return -1;
  if (cache.scalar_type() == type) return scales.has_value() ? -1 : FA_KV_CACHE_16BIT;
  if (cache.scalar_type() != at::kFloat8_e4m3fn || !scales.has_value() || !is_floats(*scales) || scales->dim() != 2 ||
      scales->size(0) != cache.size(0) || scales->size(1) != cache.size(1))
    return -1;
  return FA_KV_CACHE_E4M3;
}
bool rows_of(const Tensor &t, at::ScalarType type, std::initializer_list<int64_t> sizes) {
  return t.scalar_type() == type && t.sizes() == at::IntArrayRef(sizes.begin(), sizes.size()) && (t.size(-1) <= 1 || t.stride(-1) == 1);
}
bool all_on(const Tensor &anchor, std::initializer_list<const Tensor *> tensors, std::initializer_list<const OptTensor *> more) {
  for (const Tensor *t : tensors)
    if (!same_device(anchor, *t)) return false;
  for (const OptTensor *t : more)
    if (!same_device(anchor, *t)) return false;
  return true;
}
int32_t dtype_of(at::ScalarType type) { return type == at::kBFloat16 ? FA_DTYPE_BF16 : FA_DTYPE_F16; }
// Workspace from PyTorch's stream-ordered allocator.
struct Space {
  Tensor space;
  int64_t bytes;
  Space(int64_t need, const Tensor &like) : bytes(need) {
    if (need > 0) space = at::empty({need}, like.options().dtype(at::kByte));
  }
  void *data() const { return bytes > 0 ? space.data_ptr() : nullptr; }
};

bool append_latent(const Tensor &latent, const Tensor &rope_key, const Tensor &cache, const Tensor &block_tables, const Tensor &query_start,
                   const Tensor &context_lens, const OptTensor &norm_weight, const OptTensor &cos_sin, const OptTensor &query_rope,
                   const OptTensor &query_rope_out, const OptTensor &scales, double norm_eps, bool interleaved) {
  if (!entries.loop || !latent.is_cuda()) return false;
  if (!all_on(latent, {&rope_key, &cache, &block_tables, &query_start, &context_lens}, {&norm_weight, &cos_sin, &query_rope, &query_rope_out, &scales}))
    return false;
  const auto type = latent.scalar_type();
  if (!is_16bit(type) || latent.dim() != 2 || query_rope.has_value() != query_rope_out.has_value()) return false;
  const int32_t kind = latent_pool(cache, scales, type);
  const int64_t S = batch_of(block_tables, query_start, context_lens), T = latent.size(0);
  if (kind < 0 || S < 0 || !fits_int32(T)) return false;
  const int64_t width = cache.size(2) - kRope;
  if (!rows_of(latent, type, {T, width}) || !rows_of(rope_key, type, {T, kRope})) return false;
  fa_latent_append_shape sh = FA_LATENT_APPEND_SHAPE_INIT;
  if (query_rope.has_value()) {
    if (query_rope->dim() != 3 || !fits_int32(query_rope->size(1))) return false;
    const int64_t H = query_rope->size(1);
    if (!rows_of(*query_rope, type, {T, H, kRope}) || !rows_of(*query_rope_out, type, {T, H, kRope})) return false;
    sh.num_heads = (int32_t)H;
    sh.query_token_stride = query_rope->stride(0);
    sh.query_head_stride = query_rope->stride(1);
    sh.query_out_token_stride = query_rope_out->stride(0);
    sh.query_out_head_stride = query_rope_out->stride(1);
  }
  if (norm_weight.has_value() && (!is_floats(*norm_weight) || norm_weight->dim() != 1 || norm_weight->size(0) != width)) return false;
  if (cos_sin.has_value()) {
    if (!is_floats(*cos_sin) || cos_sin->dim() != 2 || cos_sin->size(1) != kRope || cos_sin->size(0) == 0 || !fits_int32(cos_sin->size(0))) return false;
    sh.max_positions = (int32_t)cos_sin->size(0);
  }
  sh.num_seqs = (int32_t)S;
  sh.num_tokens = (int32_t)T;
  sh.latent_dim = (int32_t)width;
  sh.rope_dim = (int32_t)kRope;
  sh.block_size = (int32_t)cache.size(1);
  sh.max_blocks_per_seq = (int32_t)block_tables.size(1);
  sh.block_stride = cache.stride(0);
  sh.token_stride = cache.stride(1);
  sh.latent_token_stride = latent.stride(0);
  sh.rope_key_token_stride = rope_key.stride(0);
  sh.src_dtype = dtype_of(type);
  sh.cache_dtype = kind;
  sh.num_pool_blocks = (int32_t)cache.size(0);
  sh.interleaved = interleaved;
  sh.norm_eps = (float)norm_eps;
  fa_paged_attention_options op = FA_PAGED_ATTENTION_OPTIONS_INIT;
  const c10::DeviceGuard guard(latent.device());
  op.stream = c10::hip::getCurrentHIPStream(latent.device().index()).stream();
  return entries.latent_append(latent.const_data_ptr(), rope_key.const_data_ptr(), cache.data_ptr(), floats(norm_weight), floats(cos_sin),
                               query_rope.has_value() ? query_rope->const_data_ptr() : nullptr,
                               query_rope_out.has_value() ? query_rope_out->data_ptr() : nullptr, const_cast<float *>(floats(scales)),
                               ints(block_tables), ints(query_start), ints(context_lens), &sh, &op) == FA_OK;
}

bool gather_latent(const Tensor &out, const Tensor &cache, const Tensor &block_tables, const Tensor &row_start, const OptTensor &first_keys,
                   const OptTensor &scales) {
  if (!entries.loop || !out.is_cuda() || !all_on(out, {&cache, &block_tables, &row_start}, {&first_keys, &scales})) return false;
  const auto type = out.scalar_type();
  const int32_t kind = is_16bit(type) ? latent_pool(cache, scales, type) : -1;
  if (kind < 0 || out.dim() != 2 || !fits_int32(out.size(0)) || !rows_of(out, type, {out.size(0), cache.size(2)})) return false;
  auto is_ints = [](const Tensor &t, int64_t dims) { return t.scalar_type() == at::kInt && t.is_contiguous() && t.dim() == dims; };
  if (!is_ints(block_tables, 2) || !is_ints(row_start, 1)) return false;
  const int64_t S = block_tables.size(0);
  if (row_start.size(0) != S + 1 || !fits_int32(S) || !fits_int32(block_tables.size(1))) return false;
  if (first_keys.has_value() && (!is_ints(*first_keys, 1) || first_keys->size(0) != S)) return false;
  fa_latent_gather_shape sh = FA_LATENT_GATHER_SHAPE_INIT;
  sh.num_seqs = (int32_t)S;
  sh.num_rows = (int32_t)out.size(0);
  sh.latent_dim = (int32_t)(cache.size(2) - kRope);
  sh.rope_dim = (int32_t)kRope;
  sh.block_size = (int32_t)cache.size(1);
  sh.max_blocks_per_seq = (int32_t)block_tables.size(1);
  sh.num_pool_blocks = (int32_t)cache.size(0);
  sh.block_stride = cache.stride(0);
  sh.token_stride = cache.stride(1);
  sh.out_stride = out.stride(0);
  sh.out_dtype = dtype_of(type);
  sh.cache_dtype = kind;
  fa_paged_attention_options op = FA_PAGED_ATTENTION_OPTIONS_INIT;
  const c10::DeviceGuard guard(out.device());
  op.stream = c10::hip::getCurrentHIPStream(out.device().index()).stream();
  return entries.latent_gather(out.data_ptr(), cache.const_data_ptr(), floats(scales), ints(block_tables), ints(row_start),
                               first_keys.has_value() ? ints(*first_keys) : nullptr, &sh, &op) == FA_OK;
}

bool attend_latent(const Tensor &out, const Tensor &query_latent, const Tensor &query_rope, const Tensor &cache, const Tensor &block_tables,
                   const Tensor &query_start, const Tensor &context_lens, double scale, int64_t most, int64_t longest, const OptTensor &scales) {
  if (!entries.loop || !query_latent.is_cuda()) return false;
  if (!all_on(query_latent, {&out, &query_rope, &cache, &block_tables, &query_start, &context_lens}, {&scales})) return false;
  const auto type = query_latent.scalar_type();
  const int32_t kind = is_16bit(type) ? latent_pool(cache, scales, type) : -1;
  const int64_t S = batch_of(block_tables, query_start, context_lens);
  if (kind < 0 || S < 0 || query_latent.dim() != 3 || !fits_int32(most) || !fits_int32(longest)) return false;
  const int64_t T = query_latent.size(0), H = query_latent.size(1), width = cache.size(2) - kRope;
  if (!fits_int32(T) || !fits_int32(H) || !rows_of(query_latent, type, {T, H, width}) || !rows_of(out, type, {T, H, width}) ||
      !rows_of(query_rope, type, {T, H, kRope}))
    return false;
  fa_latent_attention_shape sh = FA_LATENT_ATTENTION_SHAPE_INIT;
  sh.num_seqs = (int32_t)S;
  sh.num_tokens = (int32_t)T;
  sh.num_heads = (int32_t)H;
  sh.latent_dim = (int32_t)width;
  sh.rope_dim = (int32_t)kRope;
  sh.block_size = (int32_t)cache.size(1);
  sh.max_blocks_per_seq = (int32_t)block_tables.size(1);
  sh.block_stride = cache.stride(0);
  sh.token_stride = cache.stride(1);
  sh.query_latent_token_stride = query_latent.stride(0);
  sh.query_latent_head_stride = query_latent.stride(1);
  sh.query_rope_token_stride = query_rope.stride(0);
  sh.query_rope_head_stride = query_rope.stride(1);
  sh.out_token_stride = out.stride(0);
  sh.out_head_stride = out.stride(1);
  sh.q_dtype = dtype_of(type);
  sh.cache_dtype = kind;
  sh.num_pool_blocks = (int32_t)cache.size(0);
  sh.max_query_len = (int32_t)most;
  sh.max_context_len = (int32_t)longest;
  fa_paged_attention_options op = FA_PAGED_ATTENTION_OPTIONS_INIT;
  const c10::DeviceGuard guard(query_latent.device());
  op.stream = c10::hip::getCurrentHIPStream(query_latent.device().index()).stream();
  const Space space(entries.latent_workspace_bytes(&sh), query_latent);
  return entries.latent(out.data_ptr(), query_latent.const_data_ptr(), query_rope.const_data_ptr(), cache.const_data_ptr(), floats(scales),
                        ints(block_tables), ints(query_start), ints(context_lens), (float)scale, space.data(), space.bytes, &sh, &op) == FA_OK;
}

bool attend_expanded(const Tensor &out, const Tensor &query, const Tensor &key, const Tensor &rope_key, const Tensor &value,
                     const Tensor &query_start, const Tensor &key_start, double scale, int64_t most, int64_t longest) {
  if (!entries.loop || !query.is_cuda() || !all_on(query, {&out, &key, &rope_key, &value, &query_start, &key_start}, {})) return false;
  const auto type = query.scalar_type();
  if (!is_16bit(type) || query.dim() != 3 || key.dim() != 3 || !fits_int32(most) || !fits_int32(longest)) return false;
  const int64_t T = query.size(0), H = query.size(1), N = key.size(0), D = key.size(2);
  if (!fits_int32(T) || !fits_int32(H) || !fits_int32(N) || !fits_int32(D)) return false;
  if (!rows_of(query, type, {T, H, D + kRope}) || !rows_of(out, type, {T, H, D}) || !rows_of(key, type, {N, H, D}) ||
      !rows_of(value, type, {N, H, D}) || !rows_of(rope_key, type, {N, kRope}))
    return false;
  for (const Tensor *t : {&query_start, &key_start})
    if (t->scalar_type() != at::kInt || !t->is_contiguous() || t->dim() != 1 || t->size(0) < 1 || !fits_int32(t->size(0))) return false;
  if (query_start.size(0) != key_start.size(0)) return false;
  fa_latent_expanded_shape sh = FA_LATENT_EXPANDED_SHAPE_INIT;
  sh.num_seqs = (int32_t)(query_start.size(0) - 1);
  sh.num_tokens = (int32_t)T;
  sh.num_keys = (int32_t)N;
  sh.num_heads = (int32_t)H;
  sh.head_size = (int32_t)D;
  sh.rope_dim = (int32_t)kRope;
  sh.dtype = dtype_of(type);
  sh.query_token_stride = query.stride(0);
  sh.query_head_stride = query.stride(1);
  sh.key_token_stride = key.stride(0);
  sh.key_head_stride = key.stride(1);
  sh.rope_key_token_stride = rope_key.stride(0);
  sh.value_token_stride = value.stride(0);
  sh.value_head_stride = value.stride(1);
  sh.out_token_stride = out.stride(0);
  sh.out_head_stride = out.stride(1);
  sh.max_query_len = (int32_t)most;
  sh.max_key_len = (int32_t)longest;
  fa_paged_attention_options op = FA_PAGED_ATTENTION_OPTIONS_INIT;
  const c10::DeviceGuard guard(query.device());
  op.stream = c10::hip::getCurrentHIPStream(query.device().index()).stream();
  const Space space(entries.latent_expanded_workspace_bytes(&sh), query);
  return entries.latent_expanded(out.data_ptr(), query.const_data_ptr(), key.const_data_ptr(), rope_key.const_data_ptr(), value.const_data_ptr(),
                                 ints(query_start), ints(key_start), (float)scale, space.data(), space.bytes, &sh, &op) == FA_OK;
}

// ---- dispatcher kernels -------------------------------------------------------------------------
// Boxed, one for all operators: which arguments there are and which of them are written is the schema's to say.

// The operator of the same name that is written in Python.
c10::OperatorHandle in_python(const c10::OperatorHandle &op) {
  const std::string &name = op.schema().name();  // fa_amd::...
  return c10::Dispatcher::singleton().findSchemaOrThrow(("fa_amd_py" + name.substr(name.find("::"))).c_str(), "");
}

void autograd(const c10::OperatorHandle &op, c10::DispatchKeySet keys, torch::jit::Stack *stack) {
  const size_t n = op.schema().arguments().size();
  if (at::GradMode::is_enabled())
    for (const auto &arg : torch::jit::last(*stack, n))
      if (arg.isTensor() && arg.toTensor().requires_grad()) return in_python(op).callBoxed(stack);
  at::AutoDispatchBelowAutograd below;
  op.redispatchBoxed(keys & c10::after_autograd_keyset, stack);
}

void written_versions(const c10::OperatorHandle &op, c10::DispatchKeySet keys, torch::jit::Stack *stack) {
  const auto &args = op.schema().arguments();
  const auto given = torch::jit::last(*stack, args.size());
  for (size_t k = 0; k < args.size(); ++k)
    if (args[k].alias_info() && args[k].alias_info()->isWrite()) {
      if (!given[k].isTensor()) continue;  // an optional one that is not there
      const Tensor &t = given[k].toTensor();
      if (t.is_inference()) {  // (no version to count: what the Python operator says to that)
        return in_python(op).callBoxed(stack);
      }
    }
  for (size_t k = 0; k < args.size(); ++k)
    if (args[k].alias_info() && args[k].alias_info()->isWrite() && given[k].isTensor()) given[k].toTensor().unsafeGetTensorImpl()->bump_version();
  at::AutoDispatchBelowADInplaceOrView below;
  op.redispatchBoxed(keys & c10::after_ADInplaceOrView_keyset, stack);
}

// Arguments by name order of the schema; a kernel reads them off the stack, and drops them once they are launched.
struct Args {
  torch::jit::Stack *stack;
  size_t n, at = 0;
  const c10::IValue &next() { return torch::jit::peek(*stack, at++, n); }
  const Tensor &tensor() { return next().toTensor(); }
  OptTensor maybe() { return next().toOptional<Tensor>(); }
  double real() { return next().toDouble(); }
  int64_t integer() { return next().toInt(); }
};

template <bool kSplit, bool kFp8>
void attention(const c10::OperatorHandle &op, torch::jit::Stack *stack) {
  const size_t n = op.schema().arguments().size();
  Args a{stack, n};
  const Tensor &out = a.tensor();
  const Tensor *es = nullptr, *ml = nullptr, *tmp = nullptr;
  if constexpr (kSplit) es = &a.tensor(), ml = &a.tensor(), tmp = &a.tensor();
  const Tensor &query = a.tensor(), &kc = a.tensor(), &vc = a.tensor(), &tables = a.tensor(), &lens = a.tensor();
  const double scale = a.real(), fp8_scale = kFp8 ? a.real() : 1.0;
  const int64_t partition_size = kSplit ? a.integer() : 0;
  const OptTensor sinks = a.maybe(), slopes = a.maybe();
  const double softcap = a.real();
  const int64_t window_left = a.integer();
  OptTensor ks, vs;
  if constexpr (kFp8) ks = a.maybe(), vs = a.maybe();
  const int64_t longest = kSplit ? a.integer() : 0;
  bool done;
  if constexpr (kSplit) {
    const Scratch scratch{*es, *ml, *tmp};
    done = attend(out, &scratch, query, kc, vc, tables, lens, scale, kFp8, fp8_scale, partition_size, sinks, slopes, softcap,
                  window_left, ks, vs, longest);
  } else {
    done = attend(out, nullptr, query, kc, vc, tables, lens, scale, kFp8, fp8_scale, 0, sinks, slopes, softcap, window_left, ks,
                  vs, 0);
  }
  if (!done) return in_python(op).callBoxed(stack);
  torch::jit::drop(*stack, n);
}

void cache_write(const c10::OperatorHandle &op, torch::jit::Stack *stack) {
  const size_t n = op.schema().arguments().size();
  Args a{stack, n};
  const Tensor &key = a.tensor(), &value = a.tensor(), &kc = a.tensor(), &vc = a.tensor(), &slots = a.tensor();
  const double fp8_scale = a.real();
  const OptTensor ks = a.maybe(), vs = a.maybe();
  if (!append(key, value, kc, vc, slots, fp8_scale, ks, vs)) return in_python(op).callBoxed(stack);
  torch::jit::drop(*stack, n);
}

void cache_append(const c10::OperatorHandle &op, torch::jit::Stack *stack) {
  const size_t n = op.schema().arguments().size();
  Args a{stack, n};
  const Tensor &key = a.tensor(), &value = a.tensor(), &kc = a.tensor(), &vc = a.tensor(), &tables = a.tensor(), &start = a.tensor(),
               &lens = a.tensor();
  const OptTensor cos_sin = a.maybe(), query = a.maybe(), query_out = a.maybe(), ks = a.maybe(), vs = a.maybe();
  const double fp8_scale = a.real();
  const bool interleaved = a.next().toBool();
  if (!ragged_append(key, value, kc, vc, tables, start, lens, cos_sin, query, query_out, ks, vs, fp8_scale, interleaved))
    return in_python(op).callBoxed(stack);
  torch::jit::drop(*stack, n);
}

void ragged(const c10::OperatorHandle &op, torch::jit::Stack *stack) {
  const size_t n = op.schema().arguments().size();
  Args a{stack, n};
  const Tensor &out = a.tensor(), &query = a.tensor(), &kc = a.tensor(), &vc = a.tensor(), &tables = a.tensor(), &start = a.tensor(),
               &lens = a.tensor();
  const double scale = a.real();
  const int64_t most = a.integer(), longest = a.integer();
  const double fp8_scale = a.real();
  const OptTensor ks = a.maybe(), vs = a.maybe(), sinks = a.maybe(), slopes = a.maybe();
  const double softcap = a.real();
  const int64_t window_left = a.integer();
  if (!ragged_attend(out, query, kc, vc, tables, start, lens, scale, most, longest, fp8_scale, ks, vs, sinks, slopes, softcap,
                     window_left, nullptr))
    return in_python(op).callBoxed(stack);
  torch::jit::drop(*stack, n);
}

void differential(const c10::OperatorHandle &op, torch::jit::Stack *stack) {
  const size_t n = op.schema().arguments().size();
  Args a{stack, n};
  const Tensor &out = a.tensor(), &query = a.tensor(), &kc = a.tensor(), &vc = a.tensor(), &tables = a.tensor(), &start = a.tensor(),
               &lens = a.tensor();
  const double scale = a.real();
  const Tensor &lambdas = a.tensor();
  const OptTensor weight = a.maybe();
  const int64_t most = a.integer(), longest = a.integer();
  const double eps = a.real(), out_scale = a.real();
  const OptTensor ks = a.maybe(), vs = a.maybe(), none;
  const int64_t window_left = a.integer();
  const Differential diff{lambdas, weight, eps, out_scale};
  if (!ragged_attend(out, query, kc, vc, tables, start, lens, scale, most, longest, 1.0, ks, vs, none, none, 0.0, window_left, &diff))
    return in_python(op).callBoxed(stack);
  torch::jit::drop(*stack, n);
}

void latent_append(const c10::OperatorHandle &op, torch::jit::Stack *stack) {
  const size_t n = op.schema().arguments().size();
  Args a{stack, n};
  const Tensor &latent = a.tensor(), &rope_key = a.tensor(), &cache = a.tensor(), &tables = a.tensor(), &start = a.tensor(), &lens = a.tensor();
  const OptTensor weight = a.maybe(), cos_sin = a.maybe(), query = a.maybe(), query_out = a.maybe(), scales = a.maybe();
  const double eps = a.real();
  const bool interleaved = a.next().toBool();
  if (!append_latent(latent, rope_key, cache, tables, start, lens, weight, cos_sin, query, query_out, scales, eps, interleaved))
    return in_python(op).callBoxed(stack);
  torch::jit::drop(*stack, n);
}

void latent_gather(const c10::OperatorHandle &op, torch::jit::Stack *stack) {
  const size_t n = op.schema().arguments().size();
  Args a{stack, n};
  const Tensor &out = a.tensor(), &cache = a.tensor(), &tables = a.tensor(), &start = a.tensor();
  const OptTensor first = a.maybe(), scales = a.maybe();
  if (!gather_latent(out, cache, tables, start, first, scales)) return in_python(op).callBoxed(stack);
  torch::jit::drop(*stack, n);
}

void latent(const c10::OperatorHandle &op, torch::jit::Stack *stack) {
  const size_t n = op.schema().arguments().size();
  Args a{stack, n};
  const Tensor &out = a.tensor(), &query = a.tensor(), &rope = a.tensor(), &cache = a.tensor(), &tables = a.tensor(), &start = a.tensor(),
               &lens = a.tensor();
  const double scale = a.real();
  const int64_t most = a.integer(), longest = a.integer();
  const OptTensor scales = a.maybe();
  if (!attend_latent(out, query, rope, cache, tables, start, lens, scale, most, longest, scales)) return in_python(op).callBoxed(stack);
  torch::jit::drop(*stack, n);
}

void latent_expanded(const c10::OperatorHandle &op, torch::jit::Stack *stack) {
  const size_t n = op.schema().arguments().size();
  Args a{stack, n};
  const Tensor &out = a.tensor(), &query = a.tensor(), &key = a.tensor(), &rope_key = a.tensor(), &value = a.tensor(), &start = a.tensor(),
               &key_start = a.tensor();
  const double scale = a.real();
  const int64_t most = a.integer(), longest = a.integer();
  if (!attend_expanded(out, query, key, rope_key, value, start, key_start, scale, most, longest)) return in_python(op).callBoxed(stack);
  torch::jit::drop(*stack, n);
}

constexpr const char *kNames[] = {"paged_attention_loop", "paged_attention_fp8_loop", "paged_attention_reduce",
                                  "paged_attention_fp8_reduce", "kv_cache_write", "kv_cache_append", "paged_attention_ragged",
                                  "paged_attention_differential", "latent_cache_append", "latent_cache_gather",
                                  "paged_attention_latent", "attention_latent_expanded"};

}  // namespace

// table: addresses of the entry points in the order of Entries; 0: not as many as this library was built for.
extern "C" __attribute__((visibility("default"))) int fa_torch_ops_bind(void *const *table, size_t count) {
  if (count * sizeof(void *) != sizeof(Entries)) return 0;
  memcpy(&entries, table, sizeof(Entries));
  return 1;
}

extern "C" __attribute__((visibility("default"))) void fa_torch_ops_capacity_warned() { capacity_warned.store(true); }

TORCH_LIBRARY_FRAGMENT(fa_amd, m) {
  const std::vector<at::Tag> tags = {at::Tag::pt2_compliant_tag};
  m.def("paged_attention_loop(Tensor(a0!) out, Tensor query, Tensor key_cache, Tensor value_cache, Tensor block_tables, "
        "Tensor context_lens, float scale, Tensor? sinks=None, Tensor? alibi_slopes=None, float softcap=0., "
        "SymInt window_left=-1) -> ()", tags);
  m.def("paged_attention_fp8_loop(Tensor(a0!) out, Tensor query, Tensor key_cache, Tensor value_cache, Tensor block_tables, "
        "Tensor context_lens, float scale, float fp8_scale, Tensor? sinks=None, Tensor? alibi_slopes=None, float softcap=0., "
        "SymInt window_left=-1, Tensor? k_scales=None, Tensor? v_scales=None) -> ()", tags);
  m.def("paged_attention_reduce(Tensor(a0!) out, Tensor(a1!) exp_sums, Tensor(a2!) max_logits, Tensor(a3!) tmp_out, "
        "Tensor query, Tensor key_cache, Tensor value_cache, Tensor block_tables, Tensor context_lens, float scale, "
        "SymInt partition_size=0, Tensor? sinks=None, Tensor? alibi_slopes=None, float softcap=0., SymInt window_left=-1, "
        "SymInt max_context_len=-1) -> ()", tags);
  m.def("paged_attention_fp8_reduce(Tensor(a0!) out, Tensor(a1!) exp_sums, Tensor(a2!) max_logits, Tensor(a3!) tmp_out, "
        "Tensor query, Tensor key_cache, Tensor value_cache, Tensor block_tables, Tensor context_lens, float scale, "
        "float fp8_scale, SymInt partition_size=0, Tensor? sinks=None, Tensor? alibi_slopes=None, float softcap=0., "
        "SymInt window_left=-1, Tensor? k_scales=None, Tensor? v_scales=None, SymInt max_context_len=-1) -> ()", tags);
  m.def("kv_cache_write(Tensor key, Tensor value, Tensor(a2!) key_cache, Tensor(a3!) value_cache, Tensor slot_mapping, "
        "float fp8_scale=1., Tensor? k_scales=None, Tensor? v_scales=None) -> ()", tags);
  m.def("kv_cache_append(Tensor key, Tensor value, Tensor(a2!) key_cache, Tensor(a3!) value_cache, Tensor block_tables, "
        "Tensor query_start, Tensor context_lens, Tensor? cos_sin=None, Tensor? query=None, Tensor(a9!)? query_out=None, "
        "Tensor(a10!)? k_scales=None, Tensor(a11!)? v_scales=None, float fp8_scale=1., bool interleaved=False) -> ()", tags);
  m.def("paged_attention_ragged(Tensor(a0!) out, Tensor query, Tensor key_cache, Tensor value_cache, Tensor block_tables, "
        "Tensor query_start, Tensor context_lens, float scale, SymInt max_query_len, SymInt max_context_len=0, "
        "float fp8_scale=1., Tensor? k_scales=None, Tensor? v_scales=None, Tensor? sinks=None, Tensor? alibi_slopes=None, "
        "float softcap=0., SymInt window_left=-1) -> ()", tags);
  m.def("paged_attention_differential(Tensor(a0!) out, Tensor query, Tensor key_cache, Tensor value_cache, "
        "Tensor block_tables, Tensor query_start, Tensor context_lens, float scale, Tensor lambdas, Tensor? norm_weight, "
        "SymInt max_query_len, SymInt max_context_len=0, float norm_eps=1.0000000000000001e-05, float out_scale=1., "
        "Tensor? k_scales=None, Tensor? v_scales=None, SymInt window_left=-1) -> ()", tags);
  m.def("latent_cache_append(Tensor latent, Tensor rope_key, Tensor(a2!) cache, Tensor block_tables, Tensor query_start, "
        "Tensor context_lens, Tensor? norm_weight=None, Tensor? cos_sin=None, Tensor? query_rope=None, "
        "Tensor(a9!)? query_rope_out=None, Tensor(a10!)? scales=None, float norm_eps=9.9999999999999995e-07, bool interleaved=False) -> ()", tags);
  m.def("latent_cache_gather(Tensor(a0!) out, Tensor cache, Tensor block_tables, Tensor row_start, Tensor? first_keys=None, "
        "Tensor? scales=None) -> ()", tags);
  m.def("paged_attention_latent(Tensor(a0!) out, Tensor query_latent, Tensor query_rope, Tensor cache, Tensor block_tables, "
        "Tensor query_start, Tensor context_lens, float scale, SymInt max_query_len, SymInt max_context_len=0, Tensor? scales=None) -> ()", tags);
  m.def("attention_latent_expanded(Tensor(a0!) out, Tensor query, Tensor key, Tensor rope_key, Tensor value, Tensor query_start, "
        "Tensor key_start, float scale, SymInt max_query_len, SymInt max_key_len=0) -> ()", tags);
}

TORCH_LIBRARY_IMPL(fa_amd, CUDA, m) {
  m.impl("paged_attention_loop", torch::CppFunction::makeFromBoxedFunction<&attention<false, false>>());
  m.impl("paged_attention_fp8_loop", torch::CppFunction::makeFromBoxedFunction<&attention<false, true>>());
  m.impl("paged_attention_reduce", torch::CppFunction::makeFromBoxedFunction<&attention<true, false>>());
  m.impl("paged_attention_fp8_reduce", torch::CppFunction::makeFromBoxedFunction<&attention<true, true>>());
  m.impl("kv_cache_write", torch::CppFunction::makeFromBoxedFunction<&cache_write>());
  m.impl("kv_cache_append", torch::CppFunction::makeFromBoxedFunction<&cache_append>());
  m.impl("paged_attention_ragged", torch::CppFunction::makeFromBoxedFunction<&ragged>());
  m.impl("paged_attention_differential", torch::CppFunction::makeFromBoxedFunction<&differential>());
  m.impl("latent_cache_append", torch::CppFunction::makeFromBoxedFunction<&latent_append>());
  m.impl("latent_cache_gather", torch::CppFunction::makeFromBoxedFunction<&latent_gather>());
  m.impl("paged_attention_latent", torch::CppFunction::makeFromBoxedFunction<&latent>());
  m.impl("attention_latent_expanded", torch::CppFunction::makeFromBoxedFunction<&latent_expanded>());
}

TORCH_LIBRARY_IMPL(fa_amd, Autograd, m) {
  for (const char *name : kNames)
    m.impl(name, torch::CppFunction::makeFromBoxedFunction<&autograd>());
}

TORCH_LIBRARY_IMPL(fa_amd, ADInplaceOrView, m) {
  for (const char *name : kNames)
    m.impl(name, torch::CppFunction::makeFromBoxedFunction<&written_versions>());
}
