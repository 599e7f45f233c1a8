// What the kernels of ragged paged attention share: parameters, the split of the work, the two forms' common arithmetic.
//
// A row of the attention is (new token, query head[, softmax map]); the rows of one (sequence, kv head) -- new tokens times heads
// per kv head times maps -- read the same K and V.  Sequences with few rows (one new token, or a handful) go through the rows
// form (ragged_rows_kernel.h), bound by the bytes of K and V; the others through the tile form (ragged_tile_kernel.h), bound by the
// matrix cores.  Both forms may run for one call; each takes the sequences that are its own.
#pragma once

#include "kv_cache_write_kernel.h"
#include "paged_attention_wave.h"
#include "ragged_batch.h"

namespace fa {

struct RaggedParams {
  PagedAttnParams a;            // the pools, as WaveAttn addresses them
  RaggedBatch b;
  const char *query;
  char *out;
  int64_t q_token_bytes, q_head_bytes;
  const float *k_scales;        // byte pools: of (block, kv head) at [block * scale_pitch + kv head], scale_pitch 0: of kv heads
  const float *v_scales;
  int32_t scale_pitch;
  int32_t block_scales;         // scales differ from block to block
  float tensor_scale;           // byte pools without scale arrays: of V, and, but for its sign, of K
  const void *sinks;
  const float *alibi_slopes;
  float softcap;
  int32_t window;               // keys before a token's own that it sees; INT32_MAX / 2 without a window
  int32_t mask_flags;           // kMaskAlibi | kMaskSoftcap (the window is in `window`)
  float score_scale_log2;       // |scale| * log2(e)
  uint32_t query_flip;          // 0x80008000 for negative scores (scale x tensor_scale): the queries change their sign instead
  int32_t q_bf16;               // type of query and out: bf16, or fp16
  int32_t num_heads, num_kv_heads, group;
  int32_t max_query_len;
  int32_t row_limit;            // sequences with at most so many rows per kv head go through the rows form
  // differential attention
  const float *lambdas;
  const float *norm_weight;
  float norm_eps, out_scale;
  // rows form: work-groups, and their partial results
  int32_t row_groups;           // work-groups that the chip holds, at most kMaxRowGroups
  int32_t row_shares;           // shares of the line at most, each for the work-groups of all kv heads
  int32_t row_aligned;          // a work-group for each item instead: nothing is cut, nothing merged
  float *row_o;                 // [slot][16][D]
  float *row_ml;                // [slot][2][16]: maxima (base-2 units), sums
  int2 *row_seqs;               // first and last share of a sequence
  // tile form
  int32_t tile_groups;          // > 0: work-groups that share the line of tiles; 0: a work-group for each tile
  float *tile_o;                // [2 * work-group + (0: its first piece, 1: a later one)]: registers of its wavefronts
  float *tile_ml;               // [...][wavefront][2][lane]: maxima, sums
};

constexpr int kRowColumns = 16;     // rows of the rows form: MFMA columns of a wavefront
constexpr int kMaxRowGroups = 512;  // work-groups that share the line of units
constexpr int kRowUnit = 128;       // keys that a work-group of the rows form takes at a time
constexpr int kTileKeys = 64;       // keys per step of the tile form
constexpr int kNoWindow = 0x3fffffff;

// The reference that sums and weights are taken against is set kHeadroom binary orders below the maximum, and follows it only
// when it lags by more than kRefresh (every change costs a pass over the accumulators).  Probabilities reach 2^kRefresh then: within
// fp16's range, and its subnormal numbers, which round to 2^-25 whatever their size, begin at 2^-20 of the largest
// instead of 2^-14.  Sums and accumulators are 32 bits wide.
constexpr float kHeadroom = 6.0f, kRefresh = 14.0f;

// Two maps over 16-bit values: weights go to the matrix cores in two parts, the rounded ones and what the rounding left (in the tile
// form only those of bf16).  The difference of the maps, normalised, is smaller than either, and the rounding of the weights
// showed in it: with bf16 the result's error was 0.0024 of its norm, with fp16 0.00030, where rounding the result alone makes 0.0016
// and 0.0002, and two parts add nothing to that.  A single map takes one part: 0.0020 to 0.0022 with bf16, 0.00025 to 0.00028 with fp16.
template <int KVF, int MAPS>
constexpr bool two_parts() {
  return MAPS == 2 && KVF == kKv16;
}
template <typename OT>
__device__ __forceinline__ uint32_t rest_of_pair(uint32_t rounded, float lo, float hi) {
  return pack2<OT>(lo - f32_from_half_of<OT>(rounded, 0), hi - f32_from_half_of<OT>(rounded, 1));
}

// The tokens that the call has bounds for: the first max_query_len ones, and the keys that those see.
template <typename Params>
__device__ __forceinline__ RaggedSeq ragged_seq_cut(const Params &p, RaggedSeq q) {
  q.n = min(q.n, p.max_query_len);
  q.ctx = max(0, min(q.ctx, q.pos0 + q.n));
  return q;
}
template <int MAPS, typename Params>
__device__ __forceinline__ bool in_rows_form(const Params &p, const RaggedSeq &q) {
  return q.n * p.group * MAPS <= p.row_limit;
}
// Position that the j-th new token attends from: its own, or the last one that the block table has.
__device__ __forceinline__ int attends_from(const RaggedSeq &q, int j) { return min(q.pos0 + j, q.ctx - 1); }
// First key that some new token of the sequence sees.
__device__ __forceinline__ int first_key(const RaggedParams &p, const RaggedSeq &q) { return max(0, attends_from(q, 0) - p.window); }

// Units of keys that the rows form has to go through for one kv head of a sequence.
template <int MAPS>
__device__ __forceinline__ int row_units(const RaggedParams &p, RaggedSeq q) {
  q = ragged_seq_cut(p, q);
  if (q.n <= 0 || !in_rows_form<MAPS>(p, q)) return 0;
  return (q.ctx + kRowUnit - 1) / kRowUnit - first_key(p, q) / kRowUnit;
}
// Tiles of `rows` rows that the tile form has to go through for one kv head of a sequence.
template <int MAPS, int ROWS, typename Params>
__device__ __forceinline__ int row_tiles(const Params &p, RaggedSeq q) {
  q = ragged_seq_cut(p, q);
  if (q.n <= 0 || in_rows_form<MAPS>(p, q)) return 0;
  return (q.n * p.group + ROWS - 1) / ROWS;
}

// Sixteen query bits pairs, with the sign of the scale; as fp16 for byte pools.  bf16 queries are brought into fp16's range by a
// power of two of their own row (exact but for values 2^-22 and less of the row's largest): `e` is its exponent field, found by
// the caller from the largest magnitude of the whole row.
__device__ __forceinline__ uint32_t query_exponent(float largest) {
  const uint32_t e = (__builtin_bit_cast(uint32_t, largest) >> 23) & 255u;
  return min(max(e, 8u), 254u);
}
__device__ __forceinline__ u32x4 bf16_row_to_f16(u32x4 w, uint32_t e) {
  const float mul = __builtin_bit_cast(float, (261u - e) << 23);  // the row's largest value comes to lie in [2^7, 2^8)
  u32x4 o;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    o[k] = pack2<F16>(__builtin_bit_cast(float, w[k] << 16) * mul, __builtin_bit_cast(float, w[k] & 0xffff0000u) * mul);
  return o;
}
__device__ __forceinline__ float bf16_row_scale(uint32_t e) { return __builtin_bit_cast(float, (e - 7u) << 23); }
__device__ __forceinline__ float largest_of_bf16(u32x4 w, float most) {
#pragma unroll
  for (int k = 0; k < 4; ++k)
    most = fmaxf(most, fmaxf(fabsf(__builtin_bit_cast(float, w[k] << 16)), fabsf(__builtin_bit_cast(float, w[k] & 0xffff0000u))));
  return most;
}

__device__ __forceinline__ uint32_t pack_out(const RaggedParams &p, float lo, float hi) {
  return p.q_bf16 ? pack2<BF16>(lo, hi) : pack2<F16>(lo, hi);
}

// cap * tanh(x / cap) of a score in base-2 units; tanh(z) = 1 - 2 / (exp(2z) + 1)
__device__ __forceinline__ float soft_capped(float t, float cap) {
  const float e2 = fast_exp2(t * (2.0f / cap));  // exp(2 x / cap), x = t ln 2
  return cap * kLog2e * (1.0f - 2.0f * __builtin_amdgcn_rcpf(e2 + 1.0f));
}

// Sink logit of a head in base-2 units.  It joins maximum and sum at the end of a piece: as the reference of the weights, which go to
// the matrix cores in 16 bits, one far above the scores would leave them few bits.
__device__ __forceinline__ float sink_log2(const RaggedParams &p, int head) {
  return (p.q_bf16 ? load_scalar16<BF16>(reinterpret_cast<const char *>(p.sinks) + head * 2)
                   : load_scalar16<F16>(reinterpret_cast<const char *>(p.sinks) + head * 2)) * kLog2e;
}

// What a differential row with this mean square is multiplied with.  A row of zeros (a token that sees nothing) stays one without
// an epsilon, too.
__device__ __forceinline__ float norm_factor(const RaggedParams &p, float mean_square) {
  const float x = mean_square + p.norm_eps;
  return x == 0.f ? 0.f : p.out_scale / sqrtf(x);
}

// The differential result of one row from its two maps: lane l of a wavefront holds the N elements from l * N on.
template <int N>
__device__ __forceinline__ void differential_row(const RaggedParams &p, int head, int lane, const float (&o1)[N], const float (&o2)[N],
                                                 float (&x)[N]) {
  const float lambda = p.lambdas[head];
  float square = 0.f;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    x[k] = o1[k] - lambda * o2[k];
    square += x[k] * x[k];
  }
  if (p.norm_weight == nullptr) {
#pragma unroll
    for (int k = 0; k < N; ++k) x[k] *= p.out_scale;
    return;
  }
  const float mul = norm_factor(p, wave_sum(square) / (64.0f * N));
#pragma unroll
  for (int k = 0; k < N; ++k) x[k] *= mul * p.norm_weight[lane * N + k];
}

// N 16-bit elements from lane * N on of an output row.
template <int N>
__device__ __forceinline__ void store_row(const RaggedParams &p, int token, int head, int lane, const float (&x)[N]) {
  char *dst = p.out + ((int64_t)token * p.num_heads + head) * (64 * N * 2) + lane * (N * 2);
  if constexpr (N == 2) {
    *reinterpret_cast<uint32_t *>(dst) = pack_out(p, x[0], x[1]);
  } else {
    *reinterpret_cast<uint16_t *>(dst) = (uint16_t)pack_out(p, x[0], 0.f);
  }
}

}  // namespace fa
