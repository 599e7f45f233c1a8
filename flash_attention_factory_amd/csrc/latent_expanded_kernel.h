// Latent attention over expanded keys and values: causal attention of ragged batches, key = [expanded part (D), rotated part (64, shared by
// all heads)], value = D elements, a key and value head for every query head; dense arrays, the keys of the sequences one behind the other.
// Bound by the matrix cores.
//
// A work-group takes 32 tokens of one head per wavefront and goes through the keys 64 at a time.  Both parts of the keys and the
// values go from memory to LDS by themselves (loads that write LDS), into a ring of steps each, and nobody handles them on the way; the
// rotated part is a tile of its own, since it comes from another array.
//
//   S^T[key, token] = K Q^T         MFMA 32x32x16, A = keys from LDS, B = queries, in registers for good
//   online softmax                  a lane holds 32 of its token's 64 scores, lane l ^ 32 the others: one exchange per step
//   O^T[d, token]  += V^T P^T       A = values by transposing LDS reads, B = weights as the scores left them
//
// The order of the keys within the weights' k-slots is that of the score tile's registers (8 e / 4 + 4 h + e % 4 of lane half h),
// and the reads of values follow it, so weights never move between lanes.
//
// Eight wavefronts: two on each SIMD, the second four one phase behind the first, so that one is in its matrix phase while the other is in its
// vector phase.  The second four load, in their vector phase: by all, at the start of the matrix phase, the loads cost 400 to 800 cycles of
// 2300 (4096 tokens after 12288, 32 heads: 1.16 ms -> 1.04 ms).  Four wavefronts (short calls) take no turns; two such work-groups
// share a compute unit (MI355X, D = 128, 32 heads, four prompts of 1024: 67 us and 69 with eight; of 2048: 214 us and 185).
//
// With eight wavefronts the matrix cores are busy for 61 % of the time in long calls, and the clock falls to 1.6 GHz: fewer cycles
// (887 000 of once 1 116 000) have saved less time than cycles.  MI355X, over machines: 4096 tokens after 12288 0.965 to 1.02 ms (1.25 to 1.18
// PFLOP/s), six prompts of 513 to 4003 tokens 226 to 241 us (0.93 to 0.87 PFLOP/s: steps on the diagonal, start and end of a tile).
//
// Weights are rounded to the queries' type, which the matrix cores take, and their sum is that of the rounded ones: the result's error against
// 64 bits is 0.0020 to 0.0023 of its norm with bf16 and 0.00023 with fp16, where rounding the result alone makes 0.0016 and 0.0002.
#pragma once

#include "latent_absorbed_kernel.h"

namespace fa {

// Sequences whose tokens and keys lie one behind the other, with what RaggedBatch has under the same names.
struct ExpandedBatch {
  const int32_t *query_start, *key_start;  // [num_seqs + 1]
  int32_t num_seqs, num_tokens, num_keys;
  int32_t max_keys;                        // of a sequence
};
// Rows that the arrays do not have are not asked for; positions are those of the lengths as they are given, whatever has been cut.
__device__ __forceinline__ RaggedSeq expanded_seq(const ExpandedBatch &b, int32_t start, int32_t end, int32_t key_start, int32_t key_end) {
  RaggedSeq q;
  q.first = min(max(start, 0), b.num_tokens);
  const int32_t all = max(end, q.first) - q.first;
  q.n = min(all, b.num_tokens - q.first);
  const int32_t k0 = min(max(key_start, 0), b.num_keys), len = max(key_end, k0) - k0;
  q.pos0 = len - all;
  q.ctx = max(0, min(min(q.pos0 + q.n, b.max_keys), b.num_keys - k0));
  return q;
}
__device__ __forceinline__ RaggedSeq ragged_seq_uniform(const ExpandedBatch &b, int s) {
  return expanded_seq(b, load_uniform_i32(b.query_start + s), load_uniform_i32(b.query_start + s + 1), load_uniform_i32(b.key_start + s),
                      load_uniform_i32(b.key_start + s + 1));
}
__device__ __forceinline__ RaggedSeq ragged_seq_of_lane(const ExpandedBatch &b, int s) {
  return expanded_seq(b, b.query_start[s], b.query_start[s + 1], b.key_start[s], b.key_start[s + 1]);
}

struct ExpandedParams {
  ExpandedBatch b;
  const char *query, *key, *rope_key, *value;
  char *out;
  int64_t q_token_bytes, q_head_bytes, k_head_bytes, v_head_bytes, out_token_bytes, out_head_bytes;
  uint32_t k_token_bytes, r_token_bytes, v_token_bytes;
  float score_scale_log2;  // |scale| * log2(e)
  uint32_t query_flip;     // 0x80008000 for a negative scale
  int32_t max_query_len;
  // as the line of tiles knows them: a query head for each "kv head", no window, no rows form
  int32_t num_kv_heads, group, window, row_limit;
  int32_t tile_groups;     // > 0: work-groups that share the line of tiles; 0: a work-group for each tile
  float *tile_o;           // [2 * work-group + (0: its first piece, 1: a later one)]: registers of its wavefronts
  float *tile_ml;          // [...][wavefront][2][lane]: references, sums
};

template <int D, int NW>
struct ExpandedTile {
  static constexpr int kRows = NW * 32;
  static constexpr int kRing = NW == 8 ? 3 : 2;             // steps in LDS
  static constexpr int kKeyBytes = kTileKeys * D * 2, kRopeBytes = kTileKeys * kLatentRope * 2;
  static constexpr int kRopeAt = kRing * kKeyBytes, kValuesAt = kRopeAt + kRing * kRopeBytes;
  static constexpr int kLdsBytes = kValuesAt + kRing * kKeyBytes;
  static constexpr int kLoaders = 4;                        // wavefronts that load, the last ones
  static constexpr int kOwn = kTileKeys / kLoaders;         // rows of a step that one of them loads
  static constexpr int kPieces = D / 8;                     // of 16 bytes, of an expanded row
  static constexpr int kLoads = kOwn * kPieces / 64, kRopeLoads = kOwn * 8 / 64;
  static constexpr int kInFlight = 2 * kLoads + kRopeLoads;
  static_assert(kLdsBytes <= 160 * 1024 && kRows * D * 2 <= kLdsBytes, "");

  // exclusive-or of a row's pieces (the same for rows 16 apart): neither 16 rows' same piece (keys) nor 4 rows of 64 bytes (values) meet in a bank
  static __device__ __forceinline__ int key_swizzle(int key) { return D == 128 ? key & 15 : (key >> 1) & 7; }
  static __device__ __forceinline__ int rope_swizzle(int key) { return (key >> 1) & 7; }
  static __device__ __forceinline__ int value_swizzle(int key) { return D == 128 ? ((key & 3) << 2) ^ (key & 1) : ((key >> 1) & 1) * 5; }
};

// What the wavefronts of a work-group have of a tile's rows: lane (half, col) holds elements d = 32 dt + 8 k + 4 half + e of row
// `wave * 32 + col` in acc[dt][4 k + e], with the sum l.  Stores them by way of LDS, whole rows at a time.  LDS holds nothing else any more.
template <int D, typename OT>
__device__ __forceinline__ void expanded_finish(const ExpandedParams &p, const RaggedSeq &q, int head, int row0, f32x16 (&acc)[D / 32], float l,
                                                char *lds, int lane) {
  constexpr int DT = D / 32, kPer = D / 8;  // 16-byte pieces, and lanes, per row
  const int half = lane >> 5, col = lane & 31, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  char *mine = lds + wave * 32 * D * 2;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int k = 0; k < 4; ++k)
      *reinterpret_cast<u32x2 *>(mine + col * (D * 2) + (((4 * dt + k) ^ (col & (kPer - 1))) * 16) + half * 8) =
          u32x2{pack2<OT>(acc[dt][4 * k] * inv, acc[dt][4 * k + 1] * inv), pack2<OT>(acc[dt][4 * k + 2] * inv, acc[dt][4 * k + 3] * inv)};
  const int first = row0 + wave * 32, left = q.n - first;
  char *dst = p.out + (int64_t)(q.first + first) * p.out_token_bytes + head * p.out_head_bytes;
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
#pragma unroll
  for (int r0 = 0; r0 < 32; r0 += 64 / kPer) {
    const int r = r0 + lane / kPer, c = lane & (kPer - 1);
    const u32x4 v = *reinterpret_cast<const u32x4 *>(mine + r * (D * 2) + ((c ^ (r & (kPer - 1))) * 16));
    if (r < left) *reinterpret_cast<u32x4 *>(dst + r * p.out_token_bytes + c * 16) = v;
  }
}

template <int D, typename OT, int NW, bool LINE>
__global__ void __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) latent_expanded_kernel(const ExpandedParams p) {
  using T = ExpandedTile<D, NW>;
  using Line = TileLine<1, T::kRows, ExpandedParams>;
  constexpr int KS = (D + kLatentRope) / 16, DT = D / 32, R = T::kRing;
  __shared__ __attribute__((aligned(16))) char lds[T::kLdsBytes];
  const uint32_t lds_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;

  const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31, i16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool late = NW == 8 && wave >= 4, loads_here = wave >= NW - T::kLoaders;
  const int loader = wave - (NW - T::kLoaders);  // which of those that load
  const int H = p.num_kv_heads;

  // This work-group's tiles: one, longest sequences first, the last tiles of a sequence first, since they see the most keys; or a share
  // of the line.  Work-groups go to the eight XCCs in turn: tiles of one head meet in few L2 caches, either way.
  int seq, head, tile, from = 0, g = 0, end_seq = 0, end_head = 0, end_tile = 0, end_cut = 0x7fffffff;
  bool first_piece = true;
  if constexpr (LINE) {
    const Line line(p, lane);
    const int per = (line.groups + 7) >> 3;
    g = ((int)blockIdx.x & 7) * per + ((int)blockIdx.x >> 3);
    if (((int)blockIdx.x >> 3) >= per || g >= line.groups) return;
    const TilePlace at = line.find(p, line.cut(g), lane), to = line.find(p, line.cut(g + 1) - 1, lane);
    seq = at.seq, head = at.kvh, tile = at.tile;
    end_seq = to.seq, end_head = to.kvh, end_tile = to.tile;
    const RaggedSeq q0 = ragged_seq_cut(p, ragged_seq_uniform(p.b, seq)), q1 = ragged_seq_cut(p, ragged_seq_uniform(p.b, end_seq));
    const TileCosts c0 = tile_costs<1, T::kRows>(p, q0), c1 = tile_costs<1, T::kRows>(p, q1);
    from = cut_step(at.off, c0.first + c0.more * tile, tile_steps<T::kRows>(p, q0, tile).count);
    const int64_t end_cost = c1.first + c1.more * end_tile;
    const int end_count = tile_steps<T::kRows>(p, q1, end_tile).count;
    end_cut = to.off + 1 == end_cost ? end_count : cut_step(to.off + 1, end_cost, end_count);
    from = __builtin_amdgcn_readfirstlane(from), end_cut = __builtin_amdgcn_readfirstlane(end_cut);
  } else {
    const int t = blockIdx.x / H;
    head = blockIdx.x - t * H;
    int before;
    if (p.b.num_seqs <= 64) {
      const RaggedSeq mine = lane < p.b.num_seqs ? ragged_seq_of_lane(p.b, lane) : RaggedSeq{0, 0, 0, 0};
      const int tiles = lane < p.b.num_seqs ? row_tiles<1, T::kRows>(p, mine) : 0;
      before = 0;
      for (int s = 0; s < p.b.num_seqs; ++s) {
        const int ctx = __builtin_amdgcn_readlane(mine.ctx, s), n = __builtin_amdgcn_readlane(tiles, s);
        before += ctx > mine.ctx || (ctx == mine.ctx && s < lane) ? n : 0;
      }
      const unsigned long long here = __ballot(t >= before && t < before + tiles);
      if (here == 0) return;
      seq = __builtin_ctzll(here);
      before = __builtin_amdgcn_readlane(before, seq);
    } else {
      const RaggedPlace at = ragged_find(p.b.num_seqs, t, lane, [&](int s) { return row_tiles<1, T::kRows>(p, ragged_seq_of_lane(p.b, s)); });
      seq = __builtin_amdgcn_readfirstlane(at.seq);
      if (seq >= p.b.num_seqs) return;
      before = __builtin_amdgcn_readfirstlane(at.before);
    }
    tile = row_tiles<1, T::kRows>(p, ragged_seq_uniform(p.b, seq)) - 1 - (t - before);
    end_seq = seq, end_head = head, end_tile = tile;
  }
  auto meet = [&]() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
  };

  for (;; first_piece = false) {
    const RaggedSeq q = ragged_seq_cut(p, ragged_seq_uniform(p.b, seq));
    const bool last_tile = !LINE || (seq == end_seq && head == end_head && tile == end_tile);
    const int all_steps = tile_steps<T::kRows>(p, q, tile).count;
    const int until = LINE && last_tile ? min(end_cut, all_steps) : all_steps;
    const bool whole = !LINE || (from == 0 && until == all_steps);
    if (whole || from < until) {  // (a tile that sees no keys is whole: its rows get zeros)
      const int row0 = tile * T::kRows, steps = until - from;
      const int wave_row = row0 + wave * 32, row = min(wave_row + col, q.n - 1);  // rows past the end repeat the last one
      const int pos = attends_from(q, row), wave_lo = attends_from(q, min(wave_row, q.n - 1));
      const int wave_hi = attends_from(q, min(wave_row + 32, q.n) - 1);
      const int keys = attends_from(q, min(row0 + T::kRows, q.n) - 1) + 1;  // that some row of the tile sees

      u32x4 qv[KS];
      {
        const char *src = p.query + (int64_t)(q.first + row) * p.q_token_bytes + head * p.q_head_bytes + half * 16;
#pragma unroll
        for (int c = 0; c < KS; ++c) {
          qv[c] = *reinterpret_cast<const u32x4 *>(src + c * 32);
#pragma unroll
          for (int k = 0; k < 4; ++k) qv[c][k] ^= p.query_flip;
        }
      }
      float m = kNoReference, l = 0.f;
      f32x16 acc[DT];
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[dt][e] = 0.f;

      // ---- loads: a wavefront's kOwn rows of a step; of eight wavefronts the second four's, in their vector phase ----
      const int64_t k0 = min(max(load_uniform_i32(p.b.key_start + seq), 0), p.b.num_keys);
      const char *const key_rows = p.key + k0 * p.k_token_bytes + head * p.k_head_bytes;
      const char *const rope_rows = p.rope_key + k0 * p.r_token_bytes;
      const char *const value_rows = p.value + k0 * p.v_token_bytes + head * p.v_head_bytes;
      const int last_key = max(q.ctx - 1, 0);
      // Load i of a wavefront covers its rows from i * (64 / pieces) on, `kPer` lanes a row; rows past the last key repeat it.  The swizzle of
      // load i's rows is that of load 0's with `turn` * i.
      auto rows_to_lds = [&](const char *rows, uint32_t token_bytes, int key, uint32_t to, auto per, auto loads, auto turn, auto &&swizzle) __attribute__((always_inline)) {
        constexpr int kPer = decltype(per)::value, kRows = 64 / kPer;
        const int r0 = lane / kPer, piece = (lane & (kPer - 1)) ^ swizzle(r0);
        if (key + T::kOwn - 1 <= last_key) {
          const char *base = uniform_address(rows + (int64_t)key * token_bytes);
          const uint32_t row = (uint32_t)r0 * token_bytes;
#pragma unroll
          for (int i = 0; i < decltype(loads)::value; ++i)
            load_to_lds_16(__builtin_amdgcn_readfirstlane(to + i * 1024), row + (piece ^ (decltype(turn)::value * i)) * 16, base + (uint64_t)token_bytes * (i * kRows));
        } else {
          const int base_key = min(key, last_key), left = last_key - base_key;
          const char *base = uniform_address(rows + (int64_t)base_key * token_bytes);
#pragma unroll
          for (int i = 0; i < decltype(loads)::value; ++i)
            load_to_lds_16(__builtin_amdgcn_readfirstlane(to + i * 1024), (uint32_t)min(i * kRows + r0, left) * token_bytes + (piece ^ (decltype(turn)::value * i)) * 16, base);
        }
      };
      using Turn = std::integral_constant<int, 4>;
      using NoTurn = std::integral_constant<int, 0>;
      using Pieces = std::integral_constant<int, T::kPieces>;
      using Loads = std::integral_constant<int, T::kLoads>;
      auto issue_keys = [&](int n, int slot) __attribute__((always_inline)) {
        const int key = (from + n) * kTileKeys + loader * T::kOwn;
        rows_to_lds(key_rows, p.k_token_bytes, key, lds_at + slot * T::kKeyBytes + loader * T::kOwn * D * 2, Pieces{}, Loads{}, Turn{}, T::key_swizzle);
        rows_to_lds(rope_rows, p.r_token_bytes, key, lds_at + T::kRopeAt + slot * T::kRopeBytes + loader * T::kOwn * 128, std::integral_constant<int, 8>{},
                    std::integral_constant<int, T::kRopeLoads>{}, Turn{}, T::rope_swizzle);
      };
      auto issue_values = [&](int n, int slot) __attribute__((always_inline)) {
        rows_to_lds(value_rows, p.v_token_bytes, (from + n) * kTileKeys + loader * T::kOwn, lds_at + T::kValuesAt + slot * T::kKeyBytes + loader * T::kOwn * D * 2,
                    Pieces{}, Loads{}, NoTurn{}, T::value_swizzle);
      };
      // Rows that no token of the tile sees may hold anything: values of zero instead.  By the wavefront that has loaded them.
      auto clear_unseen = [&](int n, int slot) {
        const int key = (from + n) * kTileKeys + loader * T::kOwn;
        for (int r = min(max(keys - key, 0), T::kOwn); r < T::kOwn; ++r)
          if (lane < T::kPieces)
            *reinterpret_cast<u32x4 *>(lds + T::kValuesAt + slot * T::kKeyBytes + (loader * T::kOwn + r) * D * 2 + lane * 16) = u32x4{0u, 0u, 0u, 0u};
      };
      // Round n asks for the values of step n + R - 1 and the keys of n + R (the second half of eight wavefronts at the end of round n - 1,
      // beside its softmax, when nobody reads their places any more); at its end those of n + 1 and n + 2 have landed.
      int slot_k = 0, slot_v = 0;  // of keys of step n + 1, of values of step n
      auto later = [&](int slot, int by) { return slot + by >= R ? slot + by - R : slot + by; };
      auto issue = [&](int n) __attribute__((always_inline)) {
        if (n + R - 1 < steps) issue_values(n + R - 1, later(slot_v, R - 1));
        if (n + R < steps) issue_keys(n + R, later(slot_k, R - 1));
      };
      auto land = [&](int n) __attribute__((always_inline)) {
        if (n + R < steps) wait_loads<(R - 2) * T::kInFlight>();
        else wait_loads<0>();
        if (n + 1 == steps - 1) clear_unseen(n + 1, later(slot_v, 1));
      };

      // ---- the two phases of a round ----
      f32x16 x[2];  // scores of the step that softmax comes to next
      u32x4 pb[4];  // weights of the step before it, as the B operands of the values' products
      const int see_hi = wave_row < q.n && wave_hi >= 0 ? min(steps, wave_hi / kTileKeys + 1 - from) : 0;  // steps of which this wavefront sees anything
      const int k_base = col * (D * 2) + (half ^ T::key_swizzle(col)) * 16, r_base = col * 128 + (half ^ T::rope_swizzle(col)) * 16;
      const int v_key = 4 * half + (i16 >> 2);
      const int v_base = v_key * (D * 2) + ((((lane >> 4) & 1) * 2 + ((i16 & 3) >> 1)) ^ T::value_swizzle(v_key)) * 16 + (i16 & 1) * 8;
      // The matrix phase as a line of products, each with one A operand from LDS: the scores of a step (k-steps of its two halves of 32
      // keys in turn), then the values of the step before (d-tiles of its four groups of 16 keys).  kAhead operands are on
      // their way at any time; the order is held with scheduling barriers.
      constexpr int kScoreOps = 2 * KS, kValueOps = 4 * DT, kAhead = 4;
      auto operand = [&](int op, const char *kb, const char *rb, const char *vb) __attribute__((always_inline)) {
        if (op < kScoreOps) {
          const int c = op >> 1, t = op & 1;
          return c < D / 16 ? *reinterpret_cast<const u32x4 *>(kb + (k_base ^ (c << 5)) + t * 32 * 2 * D)
                            : *reinterpret_cast<const u32x4 *>(rb + (r_base ^ ((c - D / 16) << 5)) + t * 32 * 128);
        }
        const int k = (op - kScoreOps) / DT, dt = (op - kScoreOps) % DT;
        const char *at = vb + (v_base ^ (dt << 6)) + k * 16 * 2 * D;
        const u32x2 a0 = lds_read_transposed(at), a1 = lds_read_transposed(at + 8 * 2 * D);
        return u32x4{a0[0], a0[1], a1[0], a1[1]};
      };
      auto product = [&](int op, u32x4 a) __attribute__((always_inline)) {
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
      auto matrix_phase = [&](auto with_scores, auto with_values) __attribute__((always_inline)) {
        constexpr int kFirst = decltype(with_scores)::value ? 0 : kScoreOps;
        constexpr int kLast = decltype(with_values)::value ? kScoreOps + kValueOps : kScoreOps;
        const char *kb = lds + slot_k * T::kKeyBytes, *rb = lds + T::kRopeAt + slot_k * T::kRopeBytes, *vb = lds + T::kValuesAt + slot_v * T::kKeyBytes;
        u32x4 a[kAhead];
#pragma unroll
        for (int op = kFirst; op < kFirst + kAhead && op < kLast; ++op) a[(op - kFirst) % kAhead] = operand(op, kb, rb, vb);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int op = kFirst; op < kLast; ++op) {
          const int at = op - kFirst;
          product(op, a[at % kAhead]);
          if (op + kAhead < kLast) a[at % kAhead] = operand(op + kAhead, kb, rb, vb);
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      auto softmax = [&](int n) __attribute__((always_inline)) {
        const int t0 = (from + n) * kTileKeys;
        float c = p.score_scale_log2;
        // register (t, e) holds key t0 + 32 t + 8 (e / 4) + 4 half + e % 4
        if (t0 + kTileKeys - 1 > wave_lo) {
          const int hi = pos - t0 - 4 * half;
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) x[t][e] = 32 * t + 8 * (e >> 2) + (e & 3) > hi ? -INFINITY : x[t][e] * c;
          c = 1.f;
        }
        float top = max3(x[0][0], x[0][1], x[0][2]);
#pragma unroll
        for (int e = 3; e < 15; e += 2) top = max3(top, x[0][e], x[0][e + 1]);
        top = max3(top, x[0][15], x[1][0]);
#pragma unroll
        for (int e = 1; e < 15; e += 2) top = max3(top, x[1][e], x[1][e + 1]);
        top = halves_max(fmaxf(top, x[1][15])) * c;
        if (__builtin_expect(__any(top - m > kRefresh), 0)) {
          const float to = top - m > kRefresh ? top - kHeadroom : m, alpha = fast_exp2(m - to);
          l *= alpha;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) acc[dt] *= alpha;
          m = to;
        }
        float part[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const int e = (k & 1) * 8 + 2 * w;
            pb[k][w] = pack2<OT>(fast_exp2(__builtin_fmaf(x[k >> 1][e], c, -m)), fast_exp2(__builtin_fmaf(x[k >> 1][e + 1], c, -m)));
            part[w & 1] = add_pair<OT>(pb[k][w], part[w & 1]);  // the sum of the weights as they are rounded
          }
        l += part[0] + part[1];
      };

      // ---- rounds: scores of step n + 1 and values of step n, then softmax of n + 1 ----
      if (LINE && !first_piece) meet();  // LDS of the piece before has been read
      if (steps > 0) {
        constexpr bool kTurns = NW == 8;
        if (loads_here) {
          issue_keys(0, 0);
          for (int n = 0; n < R - 2; ++n) {
            if (n < steps) issue_values(n, n);
            if (n + 1 < steps) issue_keys(n + 1, n + 1);
          }
          if (R - 2 < steps) wait_loads<(R - 2) * T::kInFlight>();
          else wait_loads<0>();
          // the wait for the queries, which is one for all loads, before there are more
#pragma unroll
          for (int c = 0; c < KS; ++c) asm volatile("" : "+v"(qv[c]));
        }
        meet();
        slot_v = R - 1;  // round -1 has no values
        if (late) {
          issue(-1);
          meet();
        }
        auto advance = [&]() {
          slot_v = slot_k;
          slot_k = later(slot_k, 1);
        };
        auto before = [&](int n) __attribute__((always_inline)) {
          if (!kTurns) issue(n);
        };
        auto between = [&](int n) __attribute__((always_inline)) {  // the two phases of round n
          if (kTurns) {
            if (late) land(n);
            meet();
          }
        };
        auto after = [&](int n) __attribute__((always_inline)) {
          if (!kTurns) land(n);
          meet();
          advance();
        };
        // the loads of round n + 1: their places are those that round n + 1 has for them
        auto ask = [&](int n) __attribute__((always_inline)) {
          if (late) {
            if (n + R < steps) issue_values(n + R, slot_v);
            if (n + R + 1 < steps) issue_keys(n + R + 1, slot_k);
          }
        };
        int n = -1;
        if (see_hi > 0) {
          before(n);
          matrix_phase(std::true_type{}, std::false_type{});
          between(n);
          ask(n);
          softmax(n + 1);
          after(n);
          for (++n; n + 1 < see_hi; ++n) {
            before(n);
            if constexpr (kTurns) __builtin_amdgcn_s_setprio(1);  // products before the other half's softmax (1.05 ms -> 1.02, under the profiler)
            matrix_phase(std::true_type{}, std::true_type{});
            if constexpr (kTurns) __builtin_amdgcn_s_setprio(0);
            between(n);
            ask(n);
            softmax(n + 1);
            after(n);
          }
          before(n);
          matrix_phase(std::false_type{}, std::true_type{});
          if (n + 1 < steps) {
            between(n);
            ask(n);
            after(n);
            ++n;
          }
        }
        // rounds that the wavefront has no part in
        if (see_hi < steps)
          for (; n + 1 < steps; ++n) {
            before(n);
            between(n);
            ask(n);
            after(n);
          }
        if (kTurns && !late) meet();
      }

      // ---- results: element e of acc[dt] is d = 32 dt + 8 (e / 4) + 4 half + e % 4 of its row ----
      l = halves_sum(l);
      if (whole) {
        meet();  // nobody reads values any more
        expanded_finish<D, OT>(p, q, head, row0, acc, l, lds, LINE ? anew(lane) : lane);
      } else {
        const int64_t slot = 2 * (int64_t)g + (first_piece ? 0 : 1);
        float *dst = p.tile_o + ((slot * NW + wave) * (DT * 4) * 64 + lane) * 4;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            *reinterpret_cast<f32x4 *>(dst + (dt * 4 + k) * 256) = f32x4{acc[dt][4 * k], acc[dt][4 * k + 1], acc[dt][4 * k + 2], acc[dt][4 * k + 3]};
        float *ml = p.tile_ml + (slot * NW + wave) * 128 + lane;
        ml[0] = m;
        ml[64] = l;
      }
    }
    if (!LINE || last_tile) return;
    from = 0;
    if (++tile == row_tiles<1, T::kRows>(p, q)) {
      tile = 0;
      if (++head == H) {
        head = 0;
        do {
          if (++seq >= p.b.num_seqs) return;  // (not while the arrays stay as they are)
        } while (row_tiles<1, T::kRows>(p, ragged_seq_uniform(p.b, seq)) == 0);
      }
    }
  }
}

// Joins the pieces of a cut tile.  Work-group g looks at the cut between the shares of g and g + 1: if it is the first one within
// its tile, the pieces are those of g (its first, if its share begins with the tile, else its second one) and of the work-groups
// after it, whose first pieces they are.
template <int D, typename OT, int NW>
__global__ void __launch_bounds__(NW * 64) latent_expanded_join_kernel(const ExpandedParams p) {
  constexpr int DT = D / 32, ROWS = NW * 32;
  __shared__ __attribute__((aligned(16))) char lds[ROWS * D * 2];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const TileLine<1, ROWS, ExpandedParams> line(p, lane);
  const int g = blockIdx.x;
  if (g + 1 >= line.groups) return;
  const int64_t at = line.cut(g + 1);
  const TilePlace place = line.find(p, at, lane);
  const int64_t start = at - place.off, before = line.cut(g);  // of the tile; of the share of g
  if (place.off == 0 || before > start) return;  // a cut between two tiles, or not the first one within its tile
  const RaggedSeq q = ragged_seq_cut(p, ragged_seq_uniform(p.b, place.seq));
  const TileCosts c = tile_costs<1, ROWS>(p, q);
  const int64_t cost = c.first + c.more * place.tile;
  const int steps = tile_steps<ROWS>(p, q, place.tile).count;
  float m = kNoReference, l = 0.f;
  f32x16 acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[dt][e] = 0.f;
  int from = 0;
  for (int h = g;; ++h) {
    const int64_t share_end = h + 1 < line.groups ? line.cut(h + 1) : line.total;
    const bool last = share_end >= start + cost;
    const int until = __builtin_amdgcn_readfirstlane(last ? steps : cut_step(share_end - start, cost, steps));
    if (from == 0 && until == steps) return;  // one piece has it all: its work-group has stored the rows
    if (from < until) {
      const int64_t slot = 2 * (int64_t)h + (h == g && before < start ? 1 : 0);
      const float *ml = p.tile_ml + (slot * NW + wave) * 128 + lane;
      const float *src = p.tile_o + ((slot * NW + wave) * (DT * 4) * 64 + lane) * 4;
      const float pm = ml[0], to = fmaxf(m, pm), mine = fast_exp2(m - to), its = fast_exp2(pm - to);
      l = l * mine + ml[64] * its;
      m = to;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const f32x4 o = *reinterpret_cast<const f32x4 *>(src + (dt * 4 + k) * 256);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[dt][4 * k + e] = acc[dt][4 * k + e] * mine + o[e] * its;
        }
    }
    from = until;
    if (last) break;
  }
  expanded_finish<D, OT>(p, q, place.kvh, place.tile * ROWS, acc, l, lds, lane);
}

}  // namespace fa
