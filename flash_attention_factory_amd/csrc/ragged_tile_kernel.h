// Ragged paged attention, tile form: many rows (new token, query head) per (sequence, kv head); bound by the matrix cores.
//
// A work-group takes 32 rows per wavefront -- rows are (token, head of the kv head's group) in that order, so one pass over K and V
// serves the whole group -- and goes through the keys 64 at a time.  K and V of a step lie in LDS, both row by row as in the
// pool, in 16 bits (bytes are decoded on the way in), in two buffers: while one is computed on, the loads of the step after the
// next are in flight and the next step's are written; one barrier per step.
//
//   S^T[key, row] = K Q^T           MFMA 32x32x16, A = K from LDS (16 B per lane), B = queries, in registers for good
//   online softmax                  a lane holds 32 of its row's 64 scores, lane l ^ 32 the others: one exchange per step
//   O^T[d, row]  += V^T P^T         A = V by transposing LDS reads (ds_read_b64_tr_b16), B = P as the scores left it
//
// The order of the keys within P's k-slots is that of the score tile's registers (8 e / 4 + 4 h + e % 4 of lane half h), and the
// V reads follow it, so P never moves between lanes.  Rows of LDS are swizzled so that neither the row-wise reads of K (16 lanes,
// 16 rows, one 16-byte column) nor the transposing reads of V (32 lanes: 4 rows of 64 bytes) meet in a bank.
//
// Two maps (differential attention): half of the wavefronts take the first halves of the query and key rows, the others the second
// ones, of the same rows; V is the same; at the end the second maps' results go through LDS to the wavefronts with the first.
#pragma once

#include "ragged_attention.h"

namespace fa {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <typename OT>
__device__ __forceinline__ f32x16 mfma_32x32x16(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (std::is_same<OT, BF16>::value) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
}

// Within 16 lanes: lane 4e + c gives the address of row e's elements 4c .. 4c + 3; lane i gets element i of rows 0 .. 3.
__device__ __forceinline__ u32x2 lds_read_transposed(const char *at) {
  typedef __attribute__((address_space(3))) s16x4 *lds_ptr;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)at));
}

// The larger / the sum of the two lanes l and l ^ 32, in both.
__device__ __forceinline__ float halves_max(float v) {
  const uint32_t a = __builtin_bit_cast(uint32_t, v);
  const auto x = __builtin_amdgcn_permlane32_swap(a, a, false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)x[0]), __builtin_bit_cast(float, (uint32_t)x[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
  const uint32_t a = __builtin_bit_cast(uint32_t, v);
  const auto x = __builtin_amdgcn_permlane32_swap(a, a, false, false);
  return __builtin_bit_cast(float, (uint32_t)x[0]) + __builtin_bit_cast(float, (uint32_t)x[1]);
}

template <int D, int KVF, int MAPS, int NW>
struct RaggedTile {
  static constexpr bool KV8 = KVF != kKv16;
  static constexpr int kThreads = NW * 64;
  static constexpr int kRows = NW * 32 / MAPS;               // rows of a work-group
  static constexpr int kBufferBytes = kTileKeys * D * 2;     // K or V of a step
  static constexpr int kLdsBytes = 4 * kBufferBytes;
  static constexpr int kRowBytes = D * (KV8 ? 1 : 2);        // in the pool
  static constexpr int kPerRow = kRowBytes / 16;             // threads that load a row
  static constexpr int kRowsPerPass = kThreads / kPerRow;
  static constexpr int kPasses = kRowsPerPass >= kTileKeys ? 1 : kTileKeys / kRowsPerPass;

  // where 16-byte piece c of row `key` of a step lies in its buffer
  static __device__ __forceinline__ int k_at(int key, int c) {
    if constexpr (D == 128) return key * 256 + ((c ^ (key & 15)) * 16);
    else return key * 128 + ((c ^ ((key >> 1) & 7)) * 16);
  }
  static __device__ __forceinline__ int v_at(int key, int c) {
    if constexpr (D == 128) return key * 256 + (((c >> 2) ^ (key & 3)) * 64) + (c & 3) * 16;
    else return key * 128 + (((c >> 2) ^ ((key >> 1) & 1)) * 64) + (c & 3) * 16;
  }
};

template <int D, typename OT, int KVF, int MAPS, int NW>
__global__ void __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(2))) ragged_tile_kernel(const RaggedParams p) {
  using T = RaggedTile<D, KVF, MAPS, NW>;
  constexpr bool KV8 = T::KV8;
  constexpr int KS = D / MAPS / 16;   // k-steps of the scores
  constexpr int DT = D / 32;          // d-tiles of the output
  __shared__ __attribute__((aligned(16))) char lds[T::kLdsBytes];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5, col = lane & 31;
  const int map = MAPS == 2 ? wave / (NW / 2) : 0;
  const int strip = MAPS == 2 ? wave % (NW / 2) : wave;
  const int Hk = p.num_kv_heads, G = p.group;

  // which tile of rows: the last tiles of a sequence, which see the most keys, come first
  const int tile = blockIdx.x / Hk, kvh = blockIdx.x - tile * Hk;
  const RaggedPlace at = ragged_find(p.b.num_seqs, tile, lane,
                                     [&](int s) { return row_tiles<MAPS, T::kRows>(p, ragged_seq_of_lane(p.b, s)); });
  const int seq = __builtin_amdgcn_readfirstlane(at.seq);
  if (seq >= p.b.num_seqs) return;
  const RaggedSeq q = ragged_seq_cut(p, ragged_seq_uniform(p.b, seq));
  const int all_rows = q.n * G;
  const int row0 = (row_tiles<MAPS, T::kRows>(p, q) - 1 - (tile - __builtin_amdgcn_readfirstlane(at.before))) * T::kRows;

  // the keys that the work-group goes through, in steps of 64
  const int pos0 = q.ctx - q.n;  // position of the sequence's first new token
  const int pos_lo = pos0 + row0 / G, pos_hi = pos0 + (min(row0 + T::kRows, all_rows) - 1) / G;
  int step = max(0, pos_lo - p.window) / kTileKeys, step_end = pos_hi < 0 ? 0 : pos_hi / kTileKeys + 1;
  if (p.splits > 1) {
    const int share = (max(0, step_end - step) + p.splits - 1) / p.splits;
    step += (int)blockIdx.y * share;
    step_end = min(step_end, step + share);
  }

  // this lane's row (rows past the end repeat the last one and are not stored)
  const int my_row = row0 + strip * 32 + col;
  const bool valid = my_row < all_rows;
  const int row = min(my_row, all_rows - 1);
  const int j = row / G, head = kvh * G + (row - j * G);
  const int pos = pos0 + j;
  const int wave_row = row0 + strip * 32;
  const bool wave_live = wave_row < all_rows;
  const int wave_lo = pos0 + min(wave_row, all_rows - 1) / G, wave_hi = pos0 + (min(wave_row + 32, all_rows) - 1) / G;

  // queries: the B operand, d = 16 c + 8 half .. of the map's part
  u32x4 qv[KS];
  float q_mul = 1.f;
  {
    const char *src = p.query + (int64_t)(q.first + j) * p.q_token_bytes + head * p.q_head_bytes + map * (D / 2) * 2 + half * 16;
#pragma unroll
    for (int c = 0; c < KS; ++c) qv[c] = *reinterpret_cast<const u32x4 *>(src + c * 32);
    if (KV8 && p.q_bf16) {
      float most = 0.f;
#pragma unroll
      for (int c = 0; c < KS; ++c) most = largest_of_bf16(qv[c], most);
      const uint32_t e = query_exponent(halves_max(most));
#pragma unroll
      for (int c = 0; c < KS; ++c) qv[c] = bf16_row_to_f16(qv[c], e);
      q_mul = bf16_row_scale(e);
    }
#pragma unroll
    for (int c = 0; c < KS; ++c)
#pragma unroll
      for (int k = 0; k < 4; ++k) qv[c][k] ^= p.query_flip;
  }
  const float slope = (p.mask_flags & kMaskAlibi) ? p.alibi_slopes[head] * kLog2e : 0.f;

  float m = -INFINITY, mt = -INFINITY, l = 0.f, mv = -INFINITY, mvt = -INFINITY;
  if (p.sinks != nullptr && blockIdx.y == 0) {
    m = mt = sink_log2(p, head);
    l = half == 0 ? 1.f : 0.f;
  }
  f32x16 acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[dt][e] = 0.f;

  // ---- loads: thread (row, piece) of a step ----
  const int32_t *table = p.b.block_tables + (int64_t)seq * p.b.max_blocks_per_seq;
  const int piece = tid % T::kPerRow, load_row = tid / T::kPerRow;
  const bool loads = T::kRowsPerPass <= kTileKeys || load_row < kTileKeys;
  const int last_col = p.b.max_blocks_per_seq - 1, in_block = (1 << p.b.block_shift) - 1;
  int32_t ids[T::kPasses];
  u32x4 kreg[T::kPasses], vreg[T::kPasses];
  auto fetch_ids = [&](int st) {
#pragma unroll
    for (int x = 0; x < T::kPasses; ++x) {
      const int key = st * kTileKeys + x * T::kRowsPerPass + load_row;
      ids[x] = (int32_t)min((uint32_t)table[min(key >> p.b.block_shift, last_col)], (uint32_t)p.b.max_block_id);
    }
  };
  auto issue = [&](int st) {
    if (!loads) return;
#pragma unroll
    for (int x = 0; x < T::kPasses; ++x) {
      const int key = st * kTileKeys + x * T::kRowsPerPass + load_row;
      const int64_t off = (int64_t)ids[x] * p.a.kv_block_bytes + (int64_t)kvh * p.a.kv_head_bytes +
                          (int64_t)(key & in_block) * p.a.kv_token_bytes + piece * 16;
      kreg[x] = *reinterpret_cast<const u32x4 *>(p.a.key_cache + off);
      vreg[x] = *reinterpret_cast<const u32x4 *>(p.a.value_cache + off);
    }
  };
  auto write = [&](int st, int buf) {
    if (!loads) return;
    char *kb = lds + buf * 2 * T::kBufferBytes, *vb = kb + T::kBufferBytes;
#pragma unroll
    for (int x = 0; x < T::kPasses; ++x) {
      const int key = x * T::kRowsPerPass + load_row;
      u32x4 v = vreg[x];
      if (st * kTileKeys + key >= q.ctx) v = u32x4{0u, 0u, 0u, 0u};  // what lies there may be NaN
      if constexpr (KV8) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          u32x4 kw, vw;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            kw[w] = fp8_adjacent_pair<KVF, F16>(kreg[x][2 * h + (w >> 1)], w & 1);
            vw[w] = fp8_adjacent_pair<KVF, F16>(v[2 * h + (w >> 1)], w & 1);
          }
          *reinterpret_cast<u32x4 *>(kb + T::k_at(key, 2 * piece + h)) = kw;
          *reinterpret_cast<u32x4 *>(vb + T::v_at(key, 2 * piece + h)) = vw;
        }
      } else {
        *reinterpret_cast<u32x4 *>(kb + T::k_at(key, piece)) = kreg[x];
        *reinterpret_cast<u32x4 *>(vb + T::v_at(key, piece)) = v;
      }
    }
  };
  // scales of a step's four groups of 16 keys (a group lies within a block); groups past the context take 1
  auto fetch_scales = [&](int st, float (&sk)[4], float (&sv)[4]) {
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int key = st * kTileKeys + 16 * x;
      const int32_t id = (int32_t)min((uint32_t)load_uniform_i32(table + min(key >> p.b.block_shift, last_col)), (uint32_t)p.b.max_block_id);
      const int64_t idx = (int64_t)id * p.scale_pitch + kvh;
      const float a = load_uniform_f32(p.k_scales + idx), b = load_uniform_f32(p.v_scales + idx);
      sk[x] = key < q.ctx ? a : 1.f;
      sv[x] = key < q.ctx ? b : 1.f;
    }
  };

  if (step < step_end) {
    float sk[4] = {1.f, 1.f, 1.f, 1.f}, sv[4] = {1.f, 1.f, 1.f, 1.f}, nk[4], nv[4];
    const bool scaled = KV8 && p.k_scales != nullptr;
    const bool blocks = KV8 && p.block_scales;
    fetch_ids(step);
    issue(step);
    if (scaled) fetch_scales(step, sk, sv);
    fetch_ids(step + 1);
    write(step, 0);
    if (step + 1 < step_end) issue(step + 1);
    fetch_ids(step + 2);
    __syncthreads();
    const float c_all = p.score_scale_log2 * q_mul * (KV8 && !scaled ? p.tensor_scale : 1.f);

    for (int buf = 0; step < step_end; ++step, buf ^= 1) {
      if (scaled) fetch_scales(step + 1, nk, nv);
      const int t0 = step * kTileKeys;
      const bool sees = wave_live && t0 <= wave_hi && t0 + kTileKeys > wave_lo - p.window;  // the same for the wavefront
      if (sees) {
        const char *kb = lds + buf * 2 * T::kBufferBytes, *vb = kb + T::kBufferBytes;
        f32x16 x[2];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) x[t][e] = 0.f;
#pragma unroll
        for (int c = 0; c < KS; ++c)
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const u32x4 a = *reinterpret_cast<const u32x4 *>(kb + T::k_at(t * 32 + col, map * (D / MAPS / 8) + 2 * c + half));
            x[t] = mfma_32x32x16<OT>(a, qv[c], x[t]);
          }

        // register (t, e) holds key t0 + 32 t + 8 (e / 4) + 4 half + e % 4; group 2 t + e / 8 of 16 keys
        float cc[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) cc[k] = KV8 ? c_all * sk[k] : c_all;
        if (p.mask_flags) {  // soft-capping, distance penalties: scores in base-2 units from here on
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              float s = x[t][e] * cc[2 * t + (e >> 3)];
              if (p.mask_flags & kMaskSoftcap) s = soft_capped(s, p.softcap);
              s += slope * (float)(t0 + 32 * t + 8 * (e >> 2) + 4 * half + (e & 3) - pos);
              x[t][e] = s;
            }
#pragma unroll
          for (int k = 0; k < 4; ++k) cc[k] = 1.f;
        }
        if (t0 + kTileKeys - 1 > wave_lo || t0 < wave_hi - p.window) {
          const int hi = pos - t0 - 4 * half, lo = hi - p.window;
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const int key = 32 * t + 8 * (e >> 2) + (e & 3);
              if (key > hi || key < lo) x[t][e] = -INFINITY;  // select: the pool may hold NaN there
            }
        }
        float gm[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int t = k >> 1, e = (k & 1) * 8;
          gm[k] = fmaxf(fmaxf(fmaxf(x[t][e], x[t][e + 1]), fmaxf(x[t][e + 2], x[t][e + 3])),
                        fmaxf(fmaxf(x[t][e + 4], x[t][e + 5]), fmaxf(x[t][e + 6], x[t][e + 7]))) * cc[k];
        }
        mt = fmaxf(mt, halves_max(fmaxf(fmaxf(gm[0], gm[1]), fmaxf(gm[2], gm[3]))));
        if (__any(mt - m > kRefresh)) {
          const float to = mt - kHeadroom;
          const float alpha = m == -INFINITY ? 0.f : fast_exp2(m - to);
          l *= alpha;
          if (!blocks) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) acc[dt] *= alpha;
          }
          m = to;
        }
        const float sub = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            x[t][e] = fast_exp2(__builtin_fmaf(x[t][e], cc[2 * t + (e >> 3)], -sub));
            l += x[t][e];
          }
        float f[4];
        if (blocks) {
          float lv[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) lv[k] = __builtin_amdgcn_logf(sv[k]);
          mvt = fmaxf(mvt, halves_max(fmaxf(fmaxf(gm[0] + lv[0], gm[1] + lv[1]), fmaxf(gm[2] + lv[2], gm[3] + lv[3]))));
          if (__any(mvt - mv > kRefresh)) {
            const float to = mvt - kHeadroom;
            const float alpha = mv == -INFINITY ? 0.f : fast_exp2(mv - to);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) acc[dt] *= alpha;
            mv = to;
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) f[k] = mv == -INFINITY ? 0.f : fast_exp2(fminf(sub + lv[k] - mv, 126.0f));
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int t = k >> 1, e = (k & 1) * 8;
          u32x4 pb;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            float lo = x[t][e + 2 * w], hi = x[t][e + 2 * w + 1];
            if (blocks) {
              lo *= f[k];
              hi *= f[k];
            }
            pb[w] = pack2<OT>(lo, hi);
          }
          const int i = lane & 15, key = 16 * k + 4 * half + (i >> 2);
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) {
            const int c16 = dt * 4 + ((lane >> 4) & 1) * 2 + ((i & 3) >> 1);  // 16-byte piece; its upper 8 bytes for odd i
            const u32x2 a0 = lds_read_transposed(vb + T::v_at(key, c16) + (i & 1) * 8);
            const u32x2 a1 = lds_read_transposed(vb + T::v_at(key + 8, c16) + (i & 1) * 8);
            acc[dt] = mfma_32x32x16<OT>(u32x4{a0[0], a0[1], a1[0], a1[1]}, pb, acc[dt]);
          }
        }
      }
      if (step + 1 < step_end) {
        write(step + 1, buf ^ 1);
        if (step + 2 < step_end) issue(step + 2);
        fetch_ids(step + 3);
      }
      if (scaled) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          sk[k] = nk[k];
          sv[k] = nv[k];
        }
      }
      __syncthreads();
    }
  }

  // ---- results: element (dt, e) of a lane is d = 32 dt + 8 (e / 4) + 4 half + e % 4 of its row ----
  l = halves_sum(l);
  {
    const float to = mt == -INFINITY ? 0.f : mt;
    const float from = KV8 && p.block_scales ? mv : m;
    const float v_mul = !KV8 || p.block_scales ? 1.f : p.v_scales ? load_uniform_f32(p.v_scales + kvh) : p.tensor_scale;
    const float f = (from == -INFINITY ? 0.f : fast_exp2(from - to)) * v_mul;
    l *= m == -INFINITY ? 0.f : fast_exp2(m - to);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt] *= f;
  }
  if (p.splits > 1) {
    const int64_t slot = (int64_t)blockIdx.x * p.splits + blockIdx.y;
    const int r = map * T::kRows + strip * 32 + col;
    constexpr int kAll = T::kRows * MAPS;
    if (valid) {
      float *dst = p.tile_o + (slot * kAll + r) * D + 4 * half;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          *reinterpret_cast<f32x4 *>(dst + 32 * dt + 8 * k) = f32x4{acc[dt][4 * k], acc[dt][4 * k + 1], acc[dt][4 * k + 2], acc[dt][4 * k + 3]};
      if (half == 0) {
        p.tile_ml[slot * 2 * kAll + r] = mt;
        p.tile_ml[slot * 2 * kAll + kAll + r] = l;
      }
    }
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  char *dst = p.out + ((int64_t)(q.first + j) * p.num_heads + head) * (D * 2) + 8 * half;
  if constexpr (MAPS == 1) {
    if (valid) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          *reinterpret_cast<u32x2 *>(dst + 64 * dt + 16 * k) =
              u32x2{pack_out(p, acc[dt][4 * k] * inv, acc[dt][4 * k + 1] * inv), pack_out(p, acc[dt][4 * k + 2] * inv, acc[dt][4 * k + 3] * inv)};
    }
  } else {
    // second maps -> first maps, through LDS (a lane's values at [value][lane] of its strip); the loop's last barrier is behind
    constexpr int kValues = DT * 16;
    static_assert(kValues * 64 * 4 * (NW / 2) <= T::kLdsBytes, "the second maps' results fit the buffers");
    float *through = reinterpret_cast<float *>(lds) + strip * kValues * 64 + lane;
    if (map == 1) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) through[(dt * 16 + e) * 64] = acc[dt][e] * inv;
    }
    __syncthreads();
    if (map == 0) {
      const float lambda = p.lambdas[head];
      float square = 0.f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          acc[dt][e] = acc[dt][e] * inv - lambda * through[(dt * 16 + e) * 64];
          square += acc[dt][e] * acc[dt][e];
        }
      float mul = p.out_scale;
      if (p.norm_weight) mul /= sqrtf(halves_sum(square) / D + p.norm_eps);
      if (valid) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            f32x4 w = {mul, mul, mul, mul};
            if (p.norm_weight) w *= *reinterpret_cast<const f32x4 *>(p.norm_weight + 32 * dt + 8 * k + 4 * half);
            *reinterpret_cast<u32x2 *>(dst + 64 * dt + 16 * k) = u32x2{pack_out(p, acc[dt][4 * k] * w[0], acc[dt][4 * k + 1] * w[1]),
                                                                      pack_out(p, acc[dt][4 * k + 2] * w[2], acc[dt][4 * k + 3] * w[3])};
          }
      }
    }
  }
}

// Joins the pieces of a tile's rows: work-group (tile and kv head, 16 rows), a wavefront per row.
template <int D, int MAPS, int ROWS>
__global__ void __launch_bounds__(256) ragged_tile_merge_kernel(const RaggedParams p) {
  constexpr int N = D / 64, kAll = ROWS * MAPS;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int Hk = p.num_kv_heads, G = p.group;
  const int tile = blockIdx.x / Hk, kvh = blockIdx.x - tile * Hk;
  const RaggedPlace at = ragged_find(p.b.num_seqs, tile, lane,
                                     [&](int s) { return row_tiles<MAPS, ROWS>(p, ragged_seq_of_lane(p.b, s)); });
  const int seq = __builtin_amdgcn_readfirstlane(at.seq);
  if (seq >= p.b.num_seqs) return;
  const RaggedSeq q = ragged_seq_cut(p, ragged_seq_uniform(p.b, seq));
  const int all_rows = q.n * G;
  const int row0 = (row_tiles<MAPS, ROWS>(p, q) - 1 - (tile - __builtin_amdgcn_readfirstlane(at.before))) * ROWS;
  for (int r = (int)blockIdx.y * 16 + wave; r < (int)blockIdx.y * 16 + 16; r += 4) {
    const int row = row0 + r;
    if (row >= all_rows) return;
    const int j = row / G, head = kvh * G + (row - j * G);
    RowMerge<N> of[MAPS];
#pragma unroll
    for (int m = 0; m < MAPS; ++m) {
#pragma unroll 4
      for (int x = 0; x < p.splits; ++x) {
        const int64_t slot = (int64_t)blockIdx.x * p.splits + x;
        const float *src = p.tile_o + (slot * kAll + m * ROWS + r) * D + lane * N;
        float po[N];
#pragma unroll
        for (int k = 0; k < N; ++k) po[k] = src[k];
        of[m].add(p.tile_ml[slot * 2 * kAll + m * ROWS + r], p.tile_ml[slot * 2 * kAll + kAll + m * ROWS + r], po);
      }
      of[m].normalise();
    }
    if constexpr (MAPS == 2) {
      float x[N];
      differential_row<N>(p, head, lane, of[0].o, of[1].o, x);
      store_row<N>(p, q.first + j, head, lane, x);
    } else {
      store_row<N>(p, q.first + j, head, lane, of[0].o);
    }
  }
}

}  // namespace fa
