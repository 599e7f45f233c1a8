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

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
// c + the two 16-bit values of a dword
template <typename OT>
__device__ __forceinline__ float add_pair(uint32_t two, float c) {
  if constexpr (std::is_same<OT, BF16>::value) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, two), __builtin_bit_cast(bf16x2, 0x3f803f80u), c, false);
  } else {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, two), __builtin_bit_cast(f16x2, 0x3c003c00u), c, false);
  }
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
    if constexpr (D == 128) return key * 256 + (((c >> 2) ^ (key & 3)) * 64) + (((c & 3) ^ (key & 1)) * 16);
    else return key * 128 + (((c >> 2) ^ ((key >> 1) & 1)) * 64) + (((c & 3) ^ ((key >> 1) & 1)) * 16);
  }
};

template <int D, typename OT, int KVF, int MAPS, int NW, bool EXT>
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
  const float slope = EXT && (p.mask_flags & kMaskAlibi) ? p.alibi_slopes[head] * kLog2e : 0.f;

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
  const int steps = max(0, step_end - step);
  // Blocks of this thread's rows: of the next step of K as the table has them (cut to the pool where they are used, since
  // arithmetic here would wait for the load, and for every load before it), and of the next step of V, one step behind.
  int32_t kid[T::kPasses], vid[T::kPasses];
  u32x4 kreg[T::kPasses], vreg[T::kPasses];
  // A thread's row within its block is the same in every step, but for what a step's first key lies into a block of more than 64.
  const uint32_t block_bytes = (uint32_t)p.a.kv_block_bytes, token_bytes = (uint32_t)p.a.kv_token_bytes;
  const char *k_row[T::kPasses], *v_row[T::kPasses];
  int32_t row_col[T::kPasses];  // the thread's row in block-table columns from the step's first
#pragma unroll
  for (int x = 0; x < T::kPasses; ++x) {
    const int key = x * T::kRowsPerPass + load_row;
    const int64_t off = (int64_t)kvh * p.a.kv_head_bytes + piece * 16 + (int64_t)((uint64_t)(uint32_t)(key & in_block) * token_bytes);
    k_row[x] = p.a.key_cache + off;
    v_row[x] = p.a.value_cache + off;
    row_col[x] = key >> p.b.block_shift;
  }
  auto fetch_id = [&](int n, int x) {
    return table[(uint32_t)min(((step + n) * kTileKeys >> p.b.block_shift) + row_col[x], last_col)];
  };
  auto into_block = [&](int n) {  // bytes from the thread's row of a block's first 64 keys to its row of the step's
    return (uint64_t)(uint32_t)((step + n) * kTileKeys & in_block) * token_bytes;
  };
  // Loads past the last step are sent out like the others (the table's columns and the ids are cut, so that they read a block of
  // the pool): a condition around them would have the registers of loads in flight copied, and so waited for.
  auto issue_k = [&](int n) {
    const uint64_t more = into_block(n);
#pragma unroll
    for (int x = 0; x < T::kPasses; ++x) {
      vid[x] = (int32_t)min((uint32_t)kid[x], (uint32_t)p.b.max_block_id);
      kreg[x] = *reinterpret_cast<const u32x4 *>(k_row[x] + ((uint64_t)(uint32_t)vid[x] * block_bytes + more));
    }
#pragma unroll
    for (int x = 0; x < T::kPasses; ++x) kid[x] = fetch_id(n + 1, x);
  };
  auto issue_v = [&](int n) {  // before issue_k(n + 1)
    const uint64_t more = into_block(n);
#pragma unroll
    for (int x = 0; x < T::kPasses; ++x)
      vreg[x] = *reinterpret_cast<const u32x4 *>(v_row[x] + ((uint64_t)(uint32_t)vid[x] * block_bytes + more));
  };
  // Piece `w` of what a thread has loaded of a step, into its buffer: a 16-byte piece of LDS each.
  constexpr int kPieces = T::kPasses * (KV8 ? 2 : 1);
  auto lds_piece = [&](const u32x4 &reg, int w) {
    if constexpr (KV8) {
      u32x4 o;
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = fp8_adjacent_pair<KVF, F16>(reg[2 * (w & 1) + (k >> 1)], k & 1);
      return o;
    } else {
      return reg;
    }
  };
  auto write_k = [&](int n, int w) {
    const int pass = KV8 ? w >> 1 : w, key = pass * T::kRowsPerPass + load_row;
    const u32x4 o = lds_piece(kreg[pass], w);
    if (loads) *reinterpret_cast<u32x4 *>(lds + (n & 1) * T::kBufferBytes + T::k_at(key, KV8 ? 2 * piece + (w & 1) : piece)) = o;
  };
  auto write_v = [&](int n, int w) {
    const int pass = KV8 ? w >> 1 : w, key = pass * T::kRowsPerPass + load_row;
    if ((step + n) * kTileKeys + key >= q.ctx) vreg[pass] = u32x4{0u, 0u, 0u, 0u};  // what lies there may be NaN
    const u32x4 o = lds_piece(vreg[pass], w);
    if (loads) *reinterpret_cast<u32x4 *>(lds + (2 + (n & 1)) * T::kBufferBytes + T::v_at(key, KV8 ? 2 * piece + (w & 1) : piece)) = o;
  };
  // What a wavefront does for the coming steps during the matrix phase of step n, in small parts that lie between its products:
  // V of step n + 1 and K of n + 2 go to LDS, the loads of the step after are sent out.
  constexpr int kStageParts = 2 * kPieces + 2;
  auto stage = [&](int n, int part) {
    if (part < kPieces) write_v(n + 1, part);
    else if (part < 2 * kPieces) write_k(n + 2, part - kPieces);
    else if (part == 2 * kPieces) issue_v(n + 2);
    else if (part == 2 * kPieces + 1) issue_k(n + 3);
  };

  // Scales of a step's four groups of 16 keys (a group lies within a block): lanes 0 to 3 fetch those of K, 4 to 7 those of V, the
  // block ids two steps ahead, the scales one step ahead, both left as they come until they are used.  Groups past the context
  // take 1.
  // Byte pools without scales of blocks go the same way, with scales of 1 (log2: 0).
  constexpr bool blocks = KV8;
  const bool scaled = KV8 && p.k_scales != nullptr;
  const int group_key = 16 * (lane & 3);
  // (pools without scales: anything that can be read, not looked at, so that every step has the same loads in flight)
  const float *lane_scales = !scaled ? reinterpret_cast<const float *>(table) - kvh : (lane & 4) ? p.v_scales : p.k_scales;
  int32_t scale_id = 0;
  float scale_raw = 1.f;
  float sk[4] = {1.f, 1.f, 1.f, 1.f}, lv[4] = {0.f, 0.f, 0.f, 0.f};  // K scales and log2 of V scales of the step at hand
  auto fetch_scale_ids = [&](int n) {
    if constexpr (KV8) scale_id = table[(uint32_t)min(((step + n) * kTileKeys + group_key) >> p.b.block_shift, last_col)];
  };
  auto fetch_scales = [&]() {  // of the step that scale_id is of
    if constexpr (KV8) scale_raw = lane_scales[(int64_t)((uint64_t)min((uint32_t)scale_id, (uint32_t)p.b.max_block_id) * (uint32_t)p.scale_pitch) + kvh];
  };
  auto take_scales = [&](int n) {
    if constexpr (!KV8) return;
    const float s = scaled && (step + n) * kTileKeys + group_key < q.ctx ? scale_raw : 1.f;
    const float log = p.block_scales ? __builtin_amdgcn_logf(s) : 0.f;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      sk[x] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, s), x));
      lv[x] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, log), 4 + x));
    }
  };

  // ---- the two phases of a step ----
  const float c_all = p.score_scale_log2 * q_mul * (KV8 && !scaled ? p.tensor_scale : 1.f);
  f32x16 x[2];   // scores of the step that softmax comes to next
  u32x4 pb[4];   // weights of the step before it, as the B operands of V^T P^T
  // the steps of which this wavefront sees anything: see_lo .. see_hi - 1 (the same for all its lanes)
  const int see_lo = wave_live ? max(0, (wave_lo - p.window) / kTileKeys - step) : steps;
  const int see_hi = wave_live && wave_hi >= 0 ? min(steps, wave_hi / kTileKeys + 1 - step) : 0;
  // Where this lane reads K (16-byte piece of key `col`) and V (8 bytes of key 4 half + i / 4) within a buffer; the swizzles are
  // exclusive-ors, so a k-step or d-tile is one more of them and keys further on are an offset (see k_at, v_at).
  const int i16 = lane & 15;
  const int k_base = T::k_at(col, map * (D / MAPS / 8) + half);
  const int v_base = T::v_at(4 * half + (i16 >> 2), ((lane >> 4) & 1) * 2 + ((i16 & 3) >> 1)) + (i16 & 1) * 8;
  // The matrix phase as a line of products, each with one A operand from LDS: the scores of a step (k-steps of its two halves of 32
  // keys in turn), then the values of the step before (d-tiles of its four groups of 16 keys).  kAhead operands are on
  // their way at any time; the order is held with scheduling barriers, since left to itself the compiler reads an operand right
  // in front of the product that waits for it.
  constexpr int kScoreOps = 2 * KS, kValueOps = 4 * DT, kAhead = 6;
  auto operand = [&](int op, const char *kb, const char *vb) {
    if (op < kScoreOps) return *reinterpret_cast<const u32x4 *>(kb + (k_base ^ ((op >> 1) << 5)) + (op & 1) * 32 * 2 * D);
    const int k = (op - kScoreOps) / DT, dt = (op - kScoreOps) % DT;
    const char *at = vb + (v_base ^ (dt << 6)) + k * 16 * 2 * D;
    const u32x2 a0 = lds_read_transposed(at), a1 = lds_read_transposed(at + 8 * 2 * D);
    return u32x4{a0[0], a0[1], a1[0], a1[1]};
  };
  auto product = [&](int op, u32x4 a) {
    if (op < kScoreOps) {
      const int c = op >> 1, t = op & 1;
      if (c == 0) {
        f32x16 zero;
#pragma unroll
        for (int e = 0; e < 16; ++e) zero[e] = 0.f;
        x[t] = mfma_32x32x16<OT>(a, qv[c], zero);
      } else {
        x[t] = mfma_32x32x16<OT>(a, qv[c], x[t]);
      }
    } else {
      const int k = (op - kScoreOps) / DT, dt = (op - kScoreOps) % DT;
      acc[dt] = mfma_32x32x16<OT>(a, pb[k], acc[dt]);
    }
  };
  // scores of step n + 1 and / or values of step n
  auto matrix_phase = [&](int n, auto with_scores, auto with_values, bool with_stage) {
    constexpr int kFirst = decltype(with_scores)::value ? 0 : kScoreOps;
    constexpr int kLast = decltype(with_values)::value ? kScoreOps + kValueOps : kScoreOps;
    const char *kb = lds + ((n + 1) & 1) * T::kBufferBytes, *vb = lds + (2 + (n & 1)) * T::kBufferBytes;
    u32x4 a[kAhead];
#pragma unroll
    for (int op = kFirst; op < kFirst + kAhead && op < kLast; ++op) a[(op - kFirst) % kAhead] = operand(op, kb, vb);
    __builtin_amdgcn_sched_barrier(0);
    constexpr int kEvery = kLast - kFirst >= 2 * kStageParts + 2 ? 2 : 1;  // products from one part of the staging to the next
#pragma unroll
    for (int op = kFirst; op < kLast; ++op) {
      const int at = op - kFirst;
      product(op, a[at % kAhead]);
      if (op + kAhead < kLast) a[at % kAhead] = operand(op + kAhead, kb, vb);
      if (with_stage && at % kEvery == 0) stage(n, at / kEvery);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (with_stage) {
#pragma unroll
      for (int part = (kLast - kFirst + kEvery - 1) / kEvery; part < kStageParts; ++part) stage(n, part);
    }
  };
  auto softmax = [&](int n) {
    const int t0 = (step + n) * kTileKeys;
    // register (t, e) holds key t0 + 32 t + 8 (e / 4) + 4 half + e % 4; group 2 t + e / 8 of 16 keys
    float cc[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) cc[k] = KV8 ? c_all * sk[k] : c_all;
    if constexpr (EXT) {  // soft-capping, distance penalties: scores in base-2 units from here on
      const bool capped = p.mask_flags & kMaskSoftcap;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) x[t][e] *= cc[2 * t + (e >> 3)];
      if (capped) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) x[t][e] = soft_capped(x[t][e], p.softcap);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) x[t][e] += slope * (float)(t0 + 32 * t + 8 * (e >> 2) + 4 * half + (e & 3) - pos);
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
      gm[k] = max3(max3(max3(x[t][e], x[t][e + 1], x[t][e + 2]), x[t][e + 3], x[t][e + 4]), x[t][e + 5], x[t][e + 6]);
      gm[k] = max3(gm[k], x[t][e + 7], x[t][e + 7]);
      if constexpr (KV8) gm[k] *= cc[k];
    }
    float top = halves_max(max3(max3(gm[0], gm[1], gm[2]), gm[3], gm[3]));
    if constexpr (!KV8) top *= cc[0];
    mt = fmaxf(mt, top);
    if (__builtin_expect(__any(mt - m > kRefresh), 0)) {
      const float to = mt - kHeadroom;
      const float alpha = m == -INFINITY ? 0.f : fast_exp2(m - to);
      l *= alpha;
      if constexpr (!blocks) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[dt] *= alpha;
      }
      m = to;
    }
    const float sub = m == -INFINITY ? 0.f : m;
    if constexpr (blocks) {
      // weights 2^(score + log2(V scale) - mv); the sum takes each group's back to scores: times 2^(mv - log2(V scale) - m)
      mvt = fmaxf(mvt, halves_max(fmaxf(fmaxf(gm[0] + lv[0], gm[1] + lv[1]), fmaxf(gm[2] + lv[2], gm[3] + lv[3]))));
      if (__builtin_expect(__any(mvt - mv > kRefresh), 0)) {
        const float to = mvt - kHeadroom;
        const float alpha = mv == -INFINITY ? 0.f : fast_exp2(mv - to);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[dt] *= alpha;
        mv = to;
      }
      const float sub_v = mv == -INFINITY ? 0.f : mv;
      const float least = fminf(fminf(lv[0], lv[1]), fminf(lv[2], lv[3]));
      // A block whose V is smaller than others' by 2^80 and more (zeros, above all) would have its weights vanish, and its
      // probabilities with them: those are summed for themselves then.
      const bool apart = __any(sub_v - sub - least > 80.0f);
      if (__builtin_expect(apart, 0)) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int e = 0; e < 8; ++e) l += fast_exp2(__builtin_fmaf(x[k >> 1][(k & 1) * 8 + e], cc[k], -sub));
      }
      float part[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float from = lv[k] - sub_v;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int at = (k & 1) * 8 + e;
          x[k >> 1][at] = fast_exp2(__builtin_fmaf(x[k >> 1][at], cc[k], from));
          part[k] = e == 0 ? x[k >> 1][at] : part[k] + x[k >> 1][at];
        }
      }
      if (!apart) {
#pragma unroll
        for (int k = 0; k < 4; ++k) l = __builtin_fmaf(part[k], fast_exp2(sub_v - lv[k] - sub), l);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int at = (k & 1) * 8 + e;
          x[k >> 1][at] = fast_exp2(__builtin_fmaf(x[k >> 1][at], cc[k], -sub));
        }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int w = 0; w < 4; ++w) pb[k][w] = pack2<OT>(x[k >> 1][(k & 1) * 8 + 2 * w], x[k >> 1][(k & 1) * 8 + 2 * w + 1]);
    if constexpr (!blocks) {  // the sum of the weights as they are rounded: 16 instructions for 32 of them
      float part[2] = {0.f, 0.f};
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int w = 0; w < 4; ++w) part[w & 1] = add_pair<OT>(pb[k][w], part[w & 1]);
      l += part[0] + part[1];
    }
  };
  // Everything this work-group wrote to LDS is there, and nobody goes on before everybody is here.
  auto meet = [&]() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
  };

  // ---- steps ----
  // Matrix phase of step n: scores of n + 1 and values of n, and between the products the thread's share of V of n + 1 and K of
  // n + 2 goes to LDS (what the next matrix phase reads) and the loads of the step after that are sent out.  Vector phase: softmax
  // of n + 1.  With eight wavefronts every SIMD has two: the second four run one phase behind the first, so that one is in its
  // matrix phase while the other is in its vector phase.
  if (steps > 0) {
    constexpr bool kTurns = NW == 8;
    const int late = kTurns ? wave >> 2 : 0;
#pragma unroll
    for (int x = 0; x < T::kPasses; ++x) kid[x] = fetch_id(0, x);
    issue_k(0);
    fetch_scale_ids(0);
    fetch_scales();
    fetch_scale_ids(1);
#pragma unroll
    for (int w = 0; w < kPieces; ++w) write_k(0, w);
    issue_v(0);
    issue_k(1);
    meet();
    if (kTurns && late) meet();
    auto vector_phase = [&](int n, auto with_softmax) {
      if (kTurns) meet();
      take_scales(n + 1);
      fetch_scales();
      fetch_scale_ids(n + 3);
      if constexpr (decltype(with_softmax)::value) softmax(n + 1);
      meet();
    };
    auto idle_step = [&](int n) {
#pragma unroll
      for (int part = 0; part < kStageParts; ++part) stage(n, part);
      vector_phase(n, std::false_type{});
    };
    // Loops of their own for the steps that the wavefront has no part in, so that accumulators stay where they are.
    int n = -1;
    const int from = min(see_lo, steps), to = see_hi;
    for (; n + 1 < (from < to ? from : steps); ++n) idle_step(n);
    if (from < to) {
      matrix_phase(n, std::true_type{}, std::false_type{}, true);
      vector_phase(n, std::true_type{});
      for (++n; n + 1 < to; ++n) {
        matrix_phase(n, std::true_type{}, std::true_type{}, true);
        vector_phase(n, std::true_type{});
      }
      if (n + 1 < steps) {
        matrix_phase(n, std::false_type{}, std::true_type{}, true);
        vector_phase(n, std::false_type{});
        for (++n; n + 1 < steps; ++n) idle_step(n);
      } else {
        matrix_phase(n, std::false_type{}, std::true_type{}, false);
      }
    }
    if (kTurns && !late) meet();
  }

  // ---- results: element (dt, e) of a lane is d = 32 dt + 8 (e / 4) + 4 half + e % 4 of its row ----
  l = halves_sum(l);
  {
    const float to = mt == -INFINITY ? 0.f : mt;
    const float from = KV8 ? mv : m;
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
    // second maps -> first maps, through LDS (a lane's values at [value][lane] of its strip)
    constexpr int kValues = DT * 16;
    static_assert(kValues * 64 * 4 * (NW / 2) <= T::kLdsBytes, "the second maps' results fit the buffers");
    float *through = reinterpret_cast<float *>(lds) + strip * kValues * 64 + lane;
    __syncthreads();  // nobody reads V any more
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
