// Latent pools for gfx950: a token's row is its latent c (L elements) and its rotated key part r (64 elements), side by side, once for
// all heads.  Append: a wavefront takes a token's row -- it normalises, rotates, finds the largest magnitude, stores -- and the
// queries' rotated parts go 16 elements to a thread, as in the append of keys and values.  Gather: rows back, 16 bytes of the
// result to a thread.
//
//   c' = c * (1 / sqrt(mean c^2 + eps)) * w        in 32 bits, rounded once, when it is stored
//   r' as rotate_pair turns it
//   E4M3 pools: scale = the least power of two, 2^-100 or more, with max(|c'|, |r'|) / scale <= 448; bytes = e4m3(x / scale).  A power
//   of two leaves the values as they are, so the bytes' rounding is the only one.
//
// Bound by memory, few tokens by the launch.  MI355X: 14052 tokens of 32 heads into an FP8 pool 35 us (4.0 TB/s of what has to move); 142335 FP8
// rows back 57 us (4.3 TB/s; a device copy moves 4.8 to 5.1); one token of each of 128 sequences, 128 heads, 5.8 us.
#pragma once

#include "kv_cache_append_kernel.h"

namespace fa {

constexpr int kLatentRope = 64;  // elements of the rotated part: one for each lane of a wavefront

struct LatentAppendParams {
  KvAppendParams a;      // batch, pool and queries, as the append of keys and values has them
  const char *latent;
  const char *rope_key;
  int64_t latent_token_bytes, rope_key_token_bytes;
  const float *norm_weight;  // nullptr: latents stay as they are
  float norm_eps;
  float *scales;         // [blocks, block_size]
  int32_t row_groups;    // work-groups before those of the queries
};

// 2^e for -126 <= e <= 127
__device__ __forceinline__ float power_of_two(int e) { return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23); }

// Exponent of the scale of a row whose largest magnitude is `most`: 448 is 1.75 * 2^8.  At most 120: the reciprocal is a normal number.
__host__ __device__ __forceinline__ int row_scale_exponent(float most) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, most);
  const int e = (int)(bits >> 23) - 127 - ((bits & 0x7fffffu) <= 0x600000u ? 8 : 7);
  return e < -100 ? -100 : e;
}

template <int N, typename ST>
__device__ __forceinline__ void load_row_piece(const char *src, float (&x)[N]) {
#pragma unroll
  for (int k = 0; k < N / 4; ++k) {
    const u32x2 w = *reinterpret_cast<const u32x2 *>(src + 8 * k);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[4 * k + e] = f32_from_half_of<ST>(w[e >> 1], e & 1);
  }
}

// One row of the pool, by one wavefront: lane l has the latent's elements from l * L / 64 on, and element l of the key part.
template <int L, typename ST, bool KV8, bool INTER>
__device__ __forceinline__ void append_latent_row(const LatentAppendParams &p, int token, int seq, int32_t pos, int lane) {
  constexpr int N = L / 64;
  int32_t block = 0;
  const int64_t place = row_at(p.a, seq, pos, &block);
  if (place < 0) return;
  float x[N];
  load_row_piece<N, ST>(p.latent + token * p.latent_token_bytes + lane * (2 * N), x);
  float r = load_scalar16<ST>(p.rope_key + token * p.rope_key_token_bytes + lane * 2);
  if (p.norm_weight) {
    float square = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) square += x[k] * x[k];
    const float mul = 1.0f / sqrtf(wave_sum(square) * (1.0f / L) + p.norm_eps);
#pragma unroll
    for (int k = 0; k < N; k += 4) {
      const f32x4 w = *reinterpret_cast<const f32x4 *>(p.norm_weight + lane * N + k);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[k + e] = x[k + e] * mul * w[e];
    }
  }
  if (const float *table = angles_at(p.a, pos)) {
    const int pair = INTER ? lane >> 1 : lane & 31;
    const bool second = INTER ? lane & 1 : lane >> 5;
    const float other = __shfl_xor(r, INTER ? 1 : 32);
    float a = second ? other : r, b = second ? r : other;
    rotate_pair(a, b, table[pair], table[kLatentRope / 2 + pair]);
    r = second ? b : a;
  }
  char *dst = p.a.key_cache + place;
  if constexpr (!KV8) {
#pragma unroll
    for (int k = 0; k < N; k += 4)
      *reinterpret_cast<u32x2 *>(dst + (lane * N + k) * 2) = u32x2{pack2<ST>(x[k], x[k + 1]), pack2<ST>(x[k + 2], x[k + 3])};
    *reinterpret_cast<uint16_t *>(dst + (L + lane) * 2) = (uint16_t)pack2<ST>(r, 0.f);
  } else {
    float most = fabsf(r);
#pragma unroll
    for (int k = 0; k < N; ++k) most = fmaxf(most, fabsf(x[k]));
    const int e = row_scale_exponent(wave_max(most));
    const float mul = power_of_two(-e);
    float f[8] = {};
#pragma unroll
    for (int k = 0; k < N; ++k) f[k] = x[k] * mul;
    const u32x2 bytes = fp8_of_values<kKvE4M3>(f);
    if constexpr (N == 8) *reinterpret_cast<u32x2 *>(dst + lane * 8) = bytes;
    else *reinterpret_cast<uint32_t *>(dst + lane * 4) = bytes[0];
    const float g[8] = {r * mul, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    dst[L + lane] = (char)fp8_of_values<kKvE4M3>(g)[0];
    if (lane == 0) p.scales[((int64_t)block << p.a.b.block_shift) + (pos & ((1 << p.a.b.block_shift) - 1))] = power_of_two(e);
  }
}

template <int L, typename ST, bool KV8, bool INTER>
__global__ void __launch_bounds__(256) latent_cache_append_kernel(const LatentAppendParams p) {
  __shared__ int32_t seq[kAppendMaxTokens], pos[kAppendMaxTokens];
  if ((int)blockIdx.x < p.row_groups) {  // four rows, a wavefront each
    const int t0 = blockIdx.x * 4, count = min(4, p.a.b.num_tokens - t0);
    place_tokens(p.a.b, t0, count, seq, pos);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (wave < count && seq[wave] >= 0)
      append_latent_row<L, ST, KV8, INTER>(p, t0 + wave, __builtin_amdgcn_readfirstlane(seq[wave]), __builtin_amdgcn_readfirstlane(pos[wave]),
                                           threadIdx.x & 63);
    return;
  }
  const int t0 = ((int)blockIdx.x - p.row_groups) * p.a.tokens_per_group;
  const int count = min(p.a.tokens_per_group, p.a.b.num_tokens - t0);
  place_tokens(p.a.b, t0, count, seq, pos);
  for (int w = threadIdx.x; w < count * p.a.units_per_token; w += 256) {
    const int local = w / p.a.units_per_token, in_token = w - local * p.a.units_per_token;
    if (seq[local] >= 0) append_query_unit<ST, INTER>(p.a, t0 + local, in_token / p.a.pairs_per_row, in_token % p.a.pairs_per_row, pos[local]);
  }
}

struct LatentGatherParams {
  RaggedBatch b;             // query_start: first row of each sequence in `out`, num_tokens: rows
  const char *cache;
  const float *scales;
  const int32_t *first_keys;
  char *out;
  int64_t block_bytes, token_bytes, out_bytes;
  int32_t rows_per_group;
};
constexpr int kGatherMaxRows = 16;

template <int L, typename OT, bool KV8>
__global__ void __launch_bounds__(256) latent_cache_gather_kernel(const LatentGatherParams p) {
  constexpr int kPieces = (L + kLatentRope) / 8;  // of 8 elements
  __shared__ int64_t at[kGatherMaxRows];          // where a row lies in the pool; -1: zeros, -2: no sequence's
  __shared__ float scale[kGatherMaxRows];
  const int r0 = blockIdx.x * p.rows_per_group, count = min(p.rows_per_group, p.b.num_tokens - r0);
  if ((int)threadIdx.x < count) at[threadIdx.x] = -2;
  __syncthreads();
  for (int s = threadIdx.x; s < p.b.num_seqs; s += 256) {
    const int32_t begin = p.b.query_start[s], end = p.b.query_start[s + 1];
    const int from = max(begin, r0), to = min(end, r0 + count);
    for (int r = from; r < to; ++r) at[r - r0] = ((int64_t)s << 32) | (uint32_t)(r - begin);
  }
  __syncthreads();
  if ((int)threadIdx.x < count && at[threadIdx.x] >= 0) {
    const int s = (int)(at[threadIdx.x] >> 32);
    const int64_t key = (int64_t)(int32_t)(uint32_t)at[threadIdx.x] + (p.first_keys ? p.first_keys[s] : 0);
    int64_t row = -1;
    const int64_t col = key >> p.b.block_shift;
    if (key >= 0 && col < p.b.max_blocks_per_seq) {
      const int32_t id = p.b.block_tables[(int64_t)s * p.b.max_blocks_per_seq + col];
      const int in_block = (int)key & ((1 << p.b.block_shift) - 1);
      if ((uint32_t)id <= (uint32_t)p.b.max_block_id) {
        row = (int64_t)id * p.block_bytes + in_block * p.token_bytes;
        if constexpr (KV8) scale[threadIdx.x] = p.scales[((int64_t)id << p.b.block_shift) + in_block];
      }
    }
    at[threadIdx.x] = row;
  }
  __syncthreads();
  for (int w = threadIdx.x; w < count * kPieces; w += 256) {
    const int r = w / kPieces, c = w - r * kPieces;
    const int64_t row = at[r];
    if (row == -2) continue;
    u32x4 v = {0u, 0u, 0u, 0u};
    if (row >= 0) {
      if constexpr (KV8) {
        const u32x2 bytes = *reinterpret_cast<const u32x2 *>(p.cache + row + c * 8);
        const float s = scale[r];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const auto two = (k & 1) ? __builtin_amdgcn_cvt_pk_f32_fp8((int)bytes[k >> 1], true) : __builtin_amdgcn_cvt_pk_f32_fp8((int)bytes[k >> 1], false);
          v[k] = pack2<OT>(two[0] * s, two[1] * s);
        }
      } else {
        v = *reinterpret_cast<const u32x4 *>(p.cache + row + c * 16);
      }
    }
    *reinterpret_cast<u32x4 *>(p.out + (int64_t)(r0 + r) * p.out_bytes + c * 16) = v;
  }
}

}  // namespace fa
