// Append for gfx950: the new tokens of a ragged batch, queries and keys rotated by their positions, keys and values put into
// the paged pools at those positions.
//
// Rotation (table of cosines and sines [positions, R], R rotated elements per row): for pair k of a row at position p
//   a' = a cos(p, k) - b sin(p, k),   b' = b cos(p, k) + a sin(p, k)
// in 32 bits, each product and sum rounded by itself (no fused multiply-add: the results are those of the formula as an
// elementwise program computes it, bit for bit), rounded to the query type once, or quantised from the 32-bit value.
//
// Byte pools with a scale for each block and kv head (integers: value = byte * scale):
//   scale' = max(scale, max|x| * (1 / 127) over the new rows of the block, 2^-126), scale = 0 in a block whose first row is new;
//   rows that were there before: byte' = rint(byte * (scale / scale')), touched only where the scale grew;
//   new rows: byte = rint(x * (1 / scale')).
// One, two or four wavefronts of a work-group, by the size of a block, own the new rows of (block, kv head, K or V): they find the largest
// value, by way of LDS where they are several, and write the rows.  No atomics, and the result does not depend on the order of anything.
#pragma once

#include <type_traits>

#include "kv_cache_write_kernel.h"
#include "ragged_batch.h"

namespace fa {

struct KvAppendParams {
  RaggedBatch b;
  const char *query;       // nullptr: keys and values only
  char *query_out;
  const char *key;
  const char *value;
  char *key_cache;
  char *value_cache;
  const float *cos_sin;    // [max_positions, rotary]: cosines of the pairs, then sines; nullptr: nothing is rotated
  float *k_scales;         // per kv head (read) or per block and kv head (kept up to date)
  float *v_scales;
  int32_t scale_block_pitch;
  float inv_scale;         // 1 / fp8_scale
  int32_t max_positions;
  int32_t rotary;          // R
  int32_t num_heads;
  int32_t num_kv_heads;
  int32_t block_size;
  int64_t q_token_bytes, q_head_bytes;      // of query
  int64_t qo_token_bytes, qo_head_bytes;    // of query_out
  int64_t src_token_bytes, src_head_bytes;  // of key
  int64_t val_token_bytes, val_head_bytes;  // of value
  int64_t kv_block_bytes, kv_token_bytes, kv_head_bytes;
  // work units (kv_cache_append_kernel): threads per token and tokens per work-group
  int32_t units_per_token, tokens_per_group;
  int32_t pairs_per_row;   // units of a rotated row: 16 elements each, or 8 (see below)
  // block-scaled form: tokens that a work-group looks for block owners among, and work-groups before those of the queries
  int32_t window, kv_groups;
  int32_t team;            // wavefronts per (kv head, K or V) of an owner: 1, 2 or 4
};

constexpr float kLeastBlockScale = 1.17549435e-38f;  // 2^-126: its reciprocal is finite

template <typename ST>
__device__ __forceinline__ void unpack8(u32x4 w, float (&f)[8]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    f[2 * k] = f32_from_half_of<ST>(w[k], 0);
    f[2 * k + 1] = f32_from_half_of<ST>(w[k], 1);
  }
}
template <typename ST>
__device__ __forceinline__ u32x4 pack8(const float (&f)[8]) {
  return u32x4{pack2<ST>(f[0], f[1]), pack2<ST>(f[2], f[3]), pack2<ST>(f[4], f[5]), pack2<ST>(f[6], f[7])};
}

// One pair, every operation rounded by itself.
__device__ __forceinline__ void rotate_pair(float &a, float &b, float c, float s) {
#pragma clang fp contract(off)
  const float ac = a * c, bs = b * s, bc = b * c, as = a * s;
  a = ac - bs;
  b = bc + as;
}

// Eight elements of a row that hold four pairs of neighbours; the table row's cosines and sines of the pairs from `pair` on.
__device__ __forceinline__ void rotate_neighbours(float (&x)[8], const float *table, int half, int pair) {
  const f32x4 c = *reinterpret_cast<const f32x4 *>(table + pair), s = *reinterpret_cast<const f32x4 *>(table + half + pair);
#pragma unroll
  for (int k = 0; k < 4; ++k) rotate_pair(x[2 * k], x[2 * k + 1], c[k], s[k]);
}
// Eight pairs: x holds their first members, y the second ones.
__device__ __forceinline__ void rotate_halves(float (&x)[8], float (&y)[8], const float *table, int half, int pair) {
  const f32x4 c0 = *reinterpret_cast<const f32x4 *>(table + pair), c1 = *reinterpret_cast<const f32x4 *>(table + pair + 4);
  const f32x4 s0 = *reinterpret_cast<const f32x4 *>(table + half + pair), s1 = *reinterpret_cast<const f32x4 *>(table + half + pair + 4);
#pragma unroll
  for (int k = 0; k < 8; ++k) rotate_pair(x[k], y[k], k < 4 ? c0[k & 3] : c1[k & 3], k < 4 ? s0[k & 3] : s1[k & 3]);
}

// The two 8-element pieces of unit `u` of a row (element offsets): with pairs half the rotated elements apart, unit u of the
// rotated part is the pieces at 8u and R/2 + 8u, whose elements are partners; beyond it, and with pairs of neighbours
// everywhere, two pieces one behind the other.  (R is a multiple of 16, and so is a row.)
template <bool INTER>
__device__ __forceinline__ void unit_pieces(int u, int rotary, int &e0, int &e1) {
  const int half = rotary >> 1;
  if (!INTER && u < (half >> 3)) {
    e0 = 8 * u;
    e1 = half + 8 * u;
  } else {
    e0 = 16 * u;
    e1 = 16 * u + 8;
  }
}

template <bool INTER>
__device__ __forceinline__ void rotate_unit(float (&x)[8], float (&y)[8], int e0, const float *table, int rotary) {
  if (table == nullptr || e0 >= rotary) return;
  const int half = rotary >> 1;
  if constexpr (INTER) {
    rotate_neighbours(x, table, half, e0 >> 1);
    rotate_neighbours(y, table, half, (e0 >> 1) + 4);
  } else {
    rotate_halves(x, y, table, half, e0);
  }
}

// Row of the table for a position; a position beyond the table takes its last row (the host checks the bound it is told).
__device__ __forceinline__ const float *angles_at(const KvAppendParams &p, int32_t pos) {
  if (p.cos_sin == nullptr) return nullptr;
  return p.cos_sin + (int64_t)min(max(pos, 0), p.max_positions - 1) * p.rotary;
}

constexpr int kAppendMaxTokens = 64;  // tokens of a work-group

// Sequence and position of the work-group's tokens t0 .. t0 + count - 1 into `pos` / `seq` (LDS): every thread looks at some of the
// sequences and writes down the tokens of the group that are theirs.  -1: no sequence has the token.
__device__ __forceinline__ void place_tokens(const RaggedBatch &b, int t0, int count, int32_t *seq, int32_t *pos) {
  for (int k = threadIdx.x; k < count; k += blockDim.x) seq[k] = -1;
  __syncthreads();
  for (int s = threadIdx.x; s < b.num_seqs; s += blockDim.x) {
    const RaggedSeq q = ragged_seq_of_lane(b, s);
    const int from = max(q.first, t0), to = min(q.first + q.n, t0 + count);
    for (int t = from; t < to; ++t) {
      seq[t - t0] = s;
      pos[t - t0] = q.pos0 + (t - q.first);
    }
  }
  __syncthreads();
}

// Byte offset of a position's row of kv head 0 in the pools; -1: the position lies outside the table or its block outside the pool.
__device__ __forceinline__ int64_t row_at(const KvAppendParams &p, int seq, int32_t pos, int32_t *block) {
  if (seq < 0 || pos < 0) return -1;
  const int col = pos >> p.b.block_shift;
  if (col >= p.b.max_blocks_per_seq) return -1;
  const int32_t id = p.b.block_tables[(int64_t)seq * p.b.max_blocks_per_seq + col];
  if ((uint32_t)id > (uint32_t)p.b.max_block_id) return -1;
  *block = id;
  return (int64_t)id * p.kv_block_bytes + (int64_t)(pos & ((1 << p.b.block_shift) - 1)) * p.kv_token_bytes;
}

// One unit of a query row: load, rotate, store.
template <typename ST, bool INTER>
__device__ __forceinline__ void append_query_unit(const KvAppendParams &p, int token, int head, int u, int32_t pos) {
  int e0, e1;
  unit_pieces<INTER>(u, p.rotary, e0, e1);
  const char *src = p.query + token * p.q_token_bytes + head * p.q_head_bytes;
  char *dst = p.query_out + token * p.qo_token_bytes + head * p.qo_head_bytes;
  float x[8], y[8];
  unpack8<ST>(*reinterpret_cast<const u32x4 *>(src + 2 * e0), x);
  unpack8<ST>(*reinterpret_cast<const u32x4 *>(src + 2 * e1), y);
  rotate_unit<INTER>(x, y, e0, angles_at(p, pos), p.rotary);
  *reinterpret_cast<u32x4 *>(dst + 2 * e0) = pack8<ST>(x);
  *reinterpret_cast<u32x4 *>(dst + 2 * e1) = pack8<ST>(y);
}

// Eight values -> FP8 bytes as the tensor cast makes them (fp8_from_row_piece takes 16-bit rows; these are 32-bit values).
template <int KVF>
__device__ __forceinline__ u32x2 fp8_of_values(const float (&f)[8]) {
  u32x2 out;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t u = 0;
    if constexpr (KVF == kKvE4M3) {
      u = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[4 * h], f[4 * h + 1], 0, false);
      u = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[4 * h + 2], f[4 * h + 3], (int)u, true);
    } else {
      u = (uint32_t)__builtin_amdgcn_cvt_pk_bf8_f32(f[4 * h], f[4 * h + 1], 0, false);
      u = (uint32_t)__builtin_amdgcn_cvt_pk_bf8_f32(f[4 * h + 2], f[4 * h + 3], (int)u, true);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {  // what the cast turns into NaN, as in the writer
      const uint32_t bits = __builtin_bit_cast(uint32_t, f[4 * h + e]), mag = bits & 0x7fffffffu;
      const bool special = KVF == kKvE4M3 ? mag >= 0x43f00000u : mag > 0x7f800000u;
      if (special) u = (u & ~(0xffu << (8 * e))) | ((0x7fu | ((bits >> 24) & 0x80u)) << (8 * e));
    }
    out[h] = u;
  }
  return out;
}

// Pools of 16-bit values, and FP8 pools with given scales.  A thread takes one unit (16 elements) of one row of one token; the
// rows of a token are its query heads, the keys' kv heads, the values' kv heads.
template <typename ST, int KVF, bool INTER>
__global__ void __launch_bounds__(256) kv_cache_append_kernel(const KvAppendParams p) {
  __shared__ int32_t seq[kAppendMaxTokens], pos[kAppendMaxTokens];
  const int t0 = blockIdx.x * p.tokens_per_group;
  const int count = min(p.tokens_per_group, p.b.num_tokens - t0);
  place_tokens(p.b, t0, count, seq, pos);
  const int q_heads = p.query ? p.num_heads : 0;
  for (int w = threadIdx.x; w < count * p.units_per_token; w += 256) {
    const int local = w / p.units_per_token, in_token = w - local * p.units_per_token;
    int row = in_token / p.pairs_per_row;
    const int u = in_token - row * p.pairs_per_row;
    const int token = t0 + local;
    const int32_t at = pos[local];
    if (seq[local] < 0) continue;
    if (row < q_heads) {
      append_query_unit<ST, INTER>(p, token, row, u, at);
      continue;
    }
    row -= q_heads;
    const bool is_value = row >= p.num_kv_heads;
    const int kvh = is_value ? row - p.num_kv_heads : row;
    int32_t block = 0;
    const int64_t place = row_at(p, seq[local], at, &block);
    if (place < 0) continue;
    int e0 = 16 * u, e1 = 16 * u + 8;
    const char *src = is_value ? p.value + token * p.val_token_bytes + kvh * p.val_head_bytes
                               : p.key + token * p.src_token_bytes + kvh * p.src_head_bytes;
    char *dst = (is_value ? p.value_cache : p.key_cache) + place + kvh * p.kv_head_bytes;
    if (!is_value) unit_pieces<INTER>(u, p.rotary, e0, e1);
    const u32x4 raw0 = *reinterpret_cast<const u32x4 *>(src + 2 * e0), raw1 = *reinterpret_cast<const u32x4 *>(src + 2 * e1);
    if (KVF == kKv16 && is_value) {
      *reinterpret_cast<u32x4 *>(dst + 2 * e0) = raw0;
      *reinterpret_cast<u32x4 *>(dst + 2 * e1) = raw1;
      continue;
    }
    float x[8], y[8];
    unpack8<ST>(raw0, x);
    unpack8<ST>(raw1, y);
    if (!is_value) rotate_unit<INTER>(x, y, e0, angles_at(p, at), p.rotary);
    if constexpr (KVF == kKv16) {
      *reinterpret_cast<u32x4 *>(dst + 2 * e0) = pack8<ST>(x);
      *reinterpret_cast<u32x4 *>(dst + 2 * e1) = pack8<ST>(y);
    } else {
      const float *scales = is_value ? p.v_scales : p.k_scales;
      const float mul = scales ? 1.0f / scales[kvh] : p.inv_scale;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        x[k] *= mul;
        y[k] *= mul;
      }
      *reinterpret_cast<u32x2 *>(dst + e0) = fp8_of_values<KVF>(x);
      *reinterpret_cast<u32x2 *>(dst + e1) = fp8_of_values<KVF>(y);
    }
  }
}

// rint(x * mul) cut to -127 .. 127, eight of them as bytes; NaN becomes 0.
__device__ __forceinline__ u32x2 i8_of_values(const float (&f)[8], float mul) {
  u32x2 out = {0u, 0u};
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float t = rintf(f[k] * mul);
    const float v = t == t ? fminf(fmaxf(t, -127.0f), 127.0f) : 0.0f;
    out[k >> 2] |= ((uint32_t)(int32_t)v & 0xffu) << (8 * (k & 3));
  }
  return out;
}

// Pools of integers with a scale for each block and kv head.  Work-groups 0 .. kv_groups - 1: a window of tokens and a few
// (kv head, K or V) units; the rest: queries.  A token owns its block if it is the first of its sequence's new ones in it; the
// owner's rows are all the new ones of the block.  A unit is worked on by a team of `team` wavefronts, each with `2 * rows per
// step` rows in registers (16 of head size 128), so that blocks of up to 64 tokens are read once; larger ones are read twice.
template <typename ST, bool INTER>
__global__ void __launch_bounds__(256) kv_cache_append_scaled_kernel(const KvAppendParams p) {
  const int team = p.team;
  __shared__ int32_t seq[kAppendMaxTokens], pos[kAppendMaxTokens];
  __shared__ int32_t left[kAppendMaxTokens];  // new tokens of the sequence from this one on; 0: not an owner
  __shared__ float most_of[4];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if ((int)blockIdx.x >= p.kv_groups) {  // queries
    const int t0 = ((int)blockIdx.x - p.kv_groups) * p.tokens_per_group;
    const int count = min(p.tokens_per_group, p.b.num_tokens - t0);
    place_tokens(p.b, t0, count, seq, pos);
    for (int w = threadIdx.x; w < count * p.units_per_token; w += 256) {
      const int local = w / p.units_per_token, in_token = w - local * p.units_per_token;
      const int row = in_token / p.pairs_per_row;
      if (seq[local] >= 0) append_query_unit<ST, INTER>(p, t0 + local, row, in_token - row * p.pairs_per_row, pos[local]);
    }
    return;
  }
  const int teams = 4 / team;
  const int unit_groups = (2 * p.num_kv_heads + teams - 1) / teams;
  const int t0 = ((int)blockIdx.x / unit_groups) * p.window;
  const int unit = ((int)blockIdx.x % unit_groups) * teams + wave / team;
  const int mate = wave % team;
  const int count = min(p.window, p.b.num_tokens - t0);
  place_tokens(p.b, t0, count, seq, pos);
  for (int k = threadIdx.x; k < count; k += 256) {
    left[k] = 0;
    if (seq[k] >= 0) {
      const RaggedSeq q = ragged_seq_of_lane(p.b, seq[k]);
      const int32_t of_seq = t0 + k - q.first;
      if (of_seq == 0 || (pos[k] & (p.block_size - 1)) == 0 || pos[k] == 0) left[k] = q.n - of_seq;
    }
  }
  __syncthreads();

  const bool live = unit < 2 * p.num_kv_heads;
  const bool is_value = unit >= p.num_kv_heads;
  const int kvh = is_value ? unit - p.num_kv_heads : unit;
  const int units = p.pairs_per_row;           // 16-element units of a row
  const int per_step = 64 / units;             // rows a wavefront takes at a time
  const int lr = lane / units, u = lane - lr * units;
  int e0 = 16 * u, e1 = 16 * u + 8;
  if (!is_value) unit_pieces<INTER>(u, p.rotary, e0, e1);
  const char *src = is_value ? p.value + kvh * p.val_head_bytes : p.key + kvh * p.src_head_bytes;
  const int64_t src_token = is_value ? p.val_token_bytes : p.src_token_bytes;
  char *cache = (is_value ? p.value_cache : p.key_cache) + kvh * p.kv_head_bytes;
  float *scales = is_value ? p.v_scales : p.k_scales;

  for (int k = 0; k < count; ++k) {
    int32_t n = left[k];
    if (n == 0) continue;  // the same for the whole work-group
    const int32_t at = pos[k];
    int32_t block = 0;
    const int64_t place = row_at(p, seq[k], at, &block);
    if (place < 0) continue;  // (this, too)
    const int row0 = at & (p.block_size - 1);
    n = min(n, p.block_size - row0);
    const int64_t scale_at = (int64_t)block * p.scale_block_pitch + kvh;
    const float before = live && row0 > 0 ? scales[scale_at] : 0.0f;

    float x[2][8], y[2][8];
    auto load = [&](int first) {  // rows first .. of this wavefront's batch; rows beyond n give zeros
#pragma unroll
      for (int step = 0; step < 2; ++step) {
        const int row = first + step * per_step + lr;
        const bool ok = live && lr < per_step && row < n;
        const int64_t token = t0 + k + (ok ? row : 0);
        u32x4 a = {0u, 0u, 0u, 0u}, b = a;
        if (ok) {
          a = *reinterpret_cast<const u32x4 *>(src + token * src_token + 2 * e0);
          b = *reinterpret_cast<const u32x4 *>(src + token * src_token + 2 * e1);
        }
        unpack8<ST>(a, x[step]);
        unpack8<ST>(b, y[step]);
        if (ok && !is_value) rotate_unit<INTER>(x[step], y[step], e0, angles_at(p, at + row), p.rotary);
      }
    };
    const int batch = 2 * per_step, stride = batch * team;
    float most = 0.f;
    for (int first = mate * batch; first < n; first += stride) {
      load(first);
#pragma unroll
      for (int step = 0; step < 2; ++step)
#pragma unroll
        for (int e = 0; e < 8; ++e) most = fmaxf(most, fmaxf(fabsf(x[step][e]), fabsf(y[step][e])));
    }
    most = wave_max(most);
    if (lane == 0) most_of[wave] = most;
    __syncthreads();
    for (int w = 0; w < team; ++w) most = fmaxf(most, most_of[wave - mate + w]);
    const float after = fmaxf(fmaxf(before, most * (1.0f / 127.0f)), kLeastBlockScale);
    __syncthreads();  // (most_of is written again for the next owner)
    if (!live) continue;
    if (mate == 0 && lane == 0) scales[scale_at] = after;
    const float mul = 1.0f / after;
    char *rows = cache + place;
    const bool again = n > stride;  // the rows did not all fit the registers
    for (int first = mate * batch; first < n; first += stride) {
      if (again) load(first);
#pragma unroll
      for (int step = 0; step < 2; ++step) {
        const int row = first + step * per_step + lr;
        if (lr < per_step && row < n) {
          *reinterpret_cast<u32x2 *>(rows + row * p.kv_token_bytes + e0) = i8_of_values(x[step], mul);
          *reinterpret_cast<u32x2 *>(rows + row * p.kv_token_bytes + e1) = i8_of_values(y[step], mul);
        }
      }
    }
    if (row0 > 0 && after > before) {  // rows that were there, in the new unit
      const float ratio = before / after;
      char *old = cache + (int64_t)block * p.kv_block_bytes;
      for (int row = mate * per_step + lr; row < row0; row += team * per_step) {
        if (lr >= per_step) break;
        u32x4 *w = reinterpret_cast<u32x4 *>(old + row * p.kv_token_bytes + 16 * u);
        const u32x4 bytes = *w;
        u32x4 got;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float f[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = (float)(int8_t)(bytes[2 * h + (e >> 2)] >> (8 * (e & 3)));
          const u32x2 r = i8_of_values(f, ratio);
          got[2 * h] = r[0];
          got[2 * h + 1] = r[1];
        }
        *w = got;
      }
    }
  }
}

}  // namespace fa
