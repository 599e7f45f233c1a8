// Ragged paged attention, rows form: at most 16 rows (new token, query head, map) per (sequence, kv head), the 16 columns of an
// MFMA tile; bound by the bytes of K and V.  Measured on an MI355X: 2.0 GB of integer K and V (990 000 keys of 128 sequences, 8 kv
// heads) 341 us, 6.0 TB/s; 0.37 GB of 16-bit ones (32 sequences, 8 kv heads, two maps) 65 us, 5.7 TB/s; a single sequence of
// 30 000 keys and 4 kv heads (62 MB) 20 us, of which 5 are the two launches and 3 the second kernel.
//
// Split of the work: the keys of every sequence are cut into units of 128 and the units of all sequences are laid end to end; that
// line is cut into equal shares, whatever the lengths of the sequences are, and the work-groups of all kv heads take the same
// shares.  Those lie next to each other and go through the same blocks at the same time, whose K, V and scales lie side by side
// in the pool: shares that end at other keys from head to head took 361 us instead of 350 (and 68 instead of 65) above, and heads
// one after the other, all sequences each, up to 1.5 times as long.  A share may end within a sequence; its piece goes
// to the workspace as an unnormalised sum with its maximum (row_slot), and ragged_rows_merge_kernel joins the pieces in
// their order.  No atomics: results do not vary from run to run.
// Calls with at most 512 keys take a work-group for each (sequence, kv head) instead, without a second kernel: one sequence of 200
// keys 7.4 us and 10.7 with shares, 400 keys 9.7 and 10.7, 700 keys 12.4 and 10.5.
//
// Within a unit each of the four wavefronts takes 32 keys (WaveAttn: operands straight from the pool, no LDS) and keeps a softmax
// state of its own; the states merge through LDS at the end of a piece.
//
// Scales of the blocks of a byte pool: K's multiply the scores.  V's may not simply ride on the probabilities, which go to
// the matrix cores in 16 bits: a block of small values next to one of large ones would lose them.  So the weights have a running
// maximum of their own, mv = max(score + log2(V scale)): weight = 2^(score - m) 2^(m + log2(V scale) - mv), the second
// factor once per block, and sums and weights meet at the end, in 32 bits.
#pragma once

#include "ragged_attention.h"

namespace fa {

// Softmax state of a wavefront: column i's maximum (mt) and reference (m), sum (l); the same for the weights of V.
struct RowState {
  float m, mt, l, mv, mvt;
};

// Multipliers of a chunk's 16-key tiles.
template <int TILES>
struct RowScales {
  float k[TILES];   // raw score -> base-2 units, without the column's own factor
  float lv[TILES];  // log2 of the V scale
};

template <typename W>
struct RowColumns {
  float mul;         // what the column's raw scores are multiplied with (fp16 queries: 1)
  float slope_log2;
  int pos;           // position that the column's token attends from
  int vis_lo, vis_hi;  // keys that every column sees
  int first;         // before it: keys that no column sees
};

// Weights as operands of the matrix cores, and what their rounding left (of use with two parts, see two_parts).
template <typename W>
struct RowWeights {
  typename W::Probs top, rest;
};

template <bool KV8, bool TWO, typename W, int TILES>
__device__ __forceinline__ RowWeights<W> row_soft(W &wa, RowState &st, const RowColumns<W> &col, typename W::Chunk &R,
                                                      const typename W::Scores &s, const RowScales<TILES> &sc, int ci, int ctx,
                                                      const RaggedParams &p) {
  constexpr int NT = 4 * TILES;
  float t[NT];
#pragma unroll
  for (int e = 0; e < NT; ++e) t[e] = s.v[e >> 2][e & 3] * (sc.k[e >> 2] * col.mul);
  const int t0 = ci * W::CT;
  if (p.mask_flags & kMaskSoftcap) {
#pragma unroll
    for (int e = 0; e < NT; ++e) t[e] = soft_capped(t[e], p.softcap);
  }
  if (p.mask_flags & kMaskAlibi) {
#pragma unroll
    for (int e = 0; e < NT; ++e) t[e] += col.slope_log2 * (float)(t0 + (e >> 2) * 16 + 4 * wa.r + (e & 3) - col.pos);
  }
  if (t0 < col.vis_lo || t0 + W::CT - 1 > col.vis_hi) {  // the same for the wavefront
#pragma unroll
    for (int e = 0; e < NT; ++e) {
      const int tok = t0 + (e >> 2) * 16 + 4 * wa.r + (e & 3);
      if (tok > col.pos || tok < col.pos - p.window) t[e] = -INFINITY;  // select: the pool may hold NaN there
      if (tok >= ctx || tok < col.first) {
#pragma unroll
        for (int w = 0; w < W::VW; ++w) R.v[e][w] = 0u;
      }
    }
  }
  float mx[TILES];
#pragma unroll
  for (int h = 0; h < TILES; ++h) mx[h] = fmaxf(fmaxf(t[4 * h], t[4 * h + 1]), fmaxf(t[4 * h + 2], t[4 * h + 3]));
  float top = mx[0];
#pragma unroll
  for (int h = 1; h < TILES; ++h) top = fmaxf(top, mx[h]);
  st.mt = fmaxf(st.mt, rows_max(top));
  const bool blocks = KV8 && p.block_scales;
  if (__builtin_expect(__any(st.mt - st.m > kRefresh), 0)) {
    const float to = st.mt - kHeadroom;
    const float alpha = st.m == -INFINITY ? 0.f : fast_exp2(st.m - to);
    st.l *= alpha;
    if (!blocks) {
#pragma unroll
      for (int dt = 0; dt < W::NDT; ++dt) wa.acc[dt] *= alpha;
    }
    st.m = to;
  }
  const float sub = st.m == -INFINITY ? 0.f : st.m;
  float sum = 0.f;
#pragma unroll
  for (int e = 0; e < NT; ++e) {
    t[e] = fast_exp2(t[e] - sub);
    sum += t[e];
  }
  st.l += sum;
  if (blocks) {
    float top_v = mx[0] + sc.lv[0];
#pragma unroll
    for (int h = 1; h < TILES; ++h) top_v = fmaxf(top_v, mx[h] + sc.lv[h]);
    st.mvt = fmaxf(st.mvt, rows_max(top_v));
    if (__builtin_expect(__any(st.mvt - st.mv > kRefresh), 0)) {
      const float to = st.mvt - kHeadroom;
      const float alpha = st.mv == -INFINITY ? 0.f : fast_exp2(st.mv - to);
#pragma unroll
      for (int dt = 0; dt < W::NDT; ++dt) wa.acc[dt] *= alpha;
      st.mv = to;
    }
#pragma unroll
    for (int h = 0; h < TILES; ++h) {
      // (cut so that a weight of 0 stays 0 where the factor would overflow)
      const float f = st.mv == -INFINITY ? 0.f : fast_exp2(fminf(sub + sc.lv[h] - st.mv, 126.0f));
#pragma unroll
      for (int e = 0; e < 4; ++e) t[4 * h + e] *= f;
    }
  }
  RowWeights<W> pb;
#pragma unroll
  for (int c = 0; c < 2 * TILES; ++c) {
    const uint32_t w = pack2<typename W::Operand>(t[2 * c], t[2 * c + 1]);
    pb.top.v[c >> 2][c & 3] = w;
    if constexpr (TWO) pb.rest.v[c >> 2][c & 3] = rest_of_pair<typename W::Operand>(w, t[2 * c], t[2 * c + 1]);
  }
  return pb;
}

// Shares that the line of `total` units is cut into.  Up to 3/2 of the compute units' number, a unit each: 320 units of integers
// 11.2 us, and 13.3 with a work-group for each compute unit.  Then one for each compute unit, since pieces cost more than a second
// work-group brings, until there are 6 units for each (12 of 16-bit pools), and two from there on: 1008 units of integers 14.5 us
// with one and 15.0 with two, 1536 16.9 and 15.4, 4032 29.4 and 27.7; of 16-bit pools 940 units 19.5 and 21.3, 5800 70.8 and 68.2.
template <bool KV8>
__device__ __forceinline__ int row_shares(const RaggedParams &p, int32_t total) {
  const int64_t all = (int64_t)total * p.num_kv_heads;
  const int most = p.row_groups, half = (most + 1) >> 1;
  const int groups = all <= half + (half >> 1) || all >= (KV8 ? 6 : 12) * half ? most : half;
  return min(total, max(1, groups / p.num_kv_heads));
}
// Where a share's piece of an item lies: both sequences and shares only grow along the line, so no two pieces meet.
__device__ __forceinline__ int64_t row_slot(const RaggedParams &p, int kvh, int seq, int share) {
  return (int64_t)kvh * (p.b.num_seqs + p.row_shares) + seq + share;
}

template <int D, typename OT, int KVF, int MAPS>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) ragged_rows_kernel(const RaggedParams p) {
  constexpr bool KV8 = KVF != kKv16;
  constexpr bool kTwo = two_parts<KVF, MAPS>();
  constexpr int NW = 4;
  constexpr int TILES = 2;
  using W = WaveAttn<D, OT, KVF, TILES, Pipeline<KV8>::stream_loads_loop, false, true>;
  constexpr int NR = W::NR, NDT = W::NDT, SL = NR / NW;
  static_assert(W::CT * NW == kRowUnit, "a unit is one chunk per wavefront");
  __shared__ float lds[NW * (NR * 64 + 32)];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int Hk = p.num_kv_heads, G = p.group;

  // This work-group's share of the line of units.  The first 64 sequences' lengths are asked for once; whose turn it is
  // among them is read from the lanes.
  RaggedSeq of_lane = {0, 0, 0, 0};
  int32_t units_of_lane = 0;
  if (lane < p.b.num_seqs) {
    of_lane = ragged_seq_of_lane(p.b, lane);
    units_of_lane = row_units<MAPS>(p, of_lane);
  }
  const auto seq_at = [&](int s) {
    return s < 64 ? RaggedSeq{__builtin_amdgcn_readlane(of_lane.first, s), __builtin_amdgcn_readlane(of_lane.n, s),
                              __builtin_amdgcn_readlane(of_lane.ctx, s), __builtin_amdgcn_readlane(of_lane.pos0, s)}
                  : ragged_seq_uniform(p.b, s);
  };
  int32_t total = 0, u, u_end, before = 0;  // units of the line, this share of it, units before the sequence's own
  int shares = 0, share = 0, seq, kvh;
  if (p.row_aligned) {  // one work-group per item
    seq = blockIdx.x / Hk;
    kvh = blockIdx.x - seq * Hk;
    u = 0;
    u_end = row_units<MAPS>(p, seq_at(seq));
    const RaggedSeq q = ragged_seq_cut(p, seq_at(seq));
    if (u_end == 0) {  // no keys: zeros
      if (q.n > 0 && in_rows_form<MAPS>(p, q))
        for (int k = threadIdx.x; k < q.n * G * (D / 8); k += 256) {
          const int row = k / (D / 8), j = row / G;
          *reinterpret_cast<u32x4 *>(p.out + (((int64_t)(q.first + j) * p.num_heads + kvh * G + (row - j * G)) * D + (k % (D / 8)) * 8) * 2) =
              u32x4{0u, 0u, 0u, 0u};
        }
      return;
    }
  } else {
    const int32_t upto = wave_inclusive_scan(units_of_lane, lane);
    total = __builtin_amdgcn_readlane(upto, 63);
    if (p.b.num_seqs > 64) {
      int32_t more = 0;
      for (int s = 64 + lane; s < p.b.num_seqs; s += 64) more += row_units<MAPS>(p, ragged_seq_of_lane(p.b, s));
      total += __builtin_amdgcn_readlane(wave_inclusive_scan(more, lane), 63);
    }
    shares = row_shares<KV8>(p, total);
    share = blockIdx.x / Hk;
    kvh = blockIdx.x - share * Hk;
    if (share >= shares) return;
    u = (int32_t)((int64_t)total * share / shares);
    u_end = (int32_t)((int64_t)total * (share + 1) / shares);
    const unsigned long long beyond = __ballot(upto > u);
    if (beyond) {
      seq = __builtin_ctzll(beyond);
      before = __builtin_amdgcn_readlane(upto, seq) - __builtin_amdgcn_readlane(units_of_lane, seq);
    } else {
      const RaggedPlace at = ragged_find(p.b.num_seqs, u, lane, [&](int s) { return row_units<MAPS>(p, ragged_seq_of_lane(p.b, s)); });
      seq = __builtin_amdgcn_readfirstlane(at.seq);
      before = __builtin_amdgcn_readfirstlane(at.before);
    }
  }

  W wa(p.a, lane);
  const int r = wa.r, i = wa.i;
  do {
    // (a loop of its own, so that no way to the end of this one joins a branch on lanes: `seq` stays known to be the same for
    // the wavefront.  Where it is not, block ids and scales come with vector loads, and every one of those waits for all of K and V)
    RaggedSeq q = ragged_seq_cut(p, seq_at(seq));
    int units = row_units<MAPS>(p, q);
    while (u >= before + units && seq + 1 < p.b.num_seqs) {
      before += units;
      ++seq;
      q = ragged_seq_cut(p, seq_at(seq));
      units = row_units<MAPS>(p, q);
    }
    const int first = min(u - before, units);
    const int last = min(units, first + (u_end - u));
    u += max(last - first, 1);
    const int base_unit = first_key(p, q) / kRowUnit;
    const int tok_begin = (base_unit + first) * kRowUnit, tok_end = min(q.ctx, (base_unit + last) * kRowUnit);
    const int32_t *table = p.b.block_tables + (int64_t)seq * p.b.max_blocks_per_seq;
    const int last_col = p.b.max_blocks_per_seq - 1;
    int ci = tok_begin / W::CT + wave;
    const int c_end = (tok_end + W::CT - 1) / W::CT;

    // block scales of a chunk; tiles that no column sees take 1, whatever the block that their id names holds
    auto fetch_scales = [&](const typename W::Ids &ids, int c) {
      RowScales<TILES> x;
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        x.k[t] = p.score_scale_log2;
        x.lv[t] = 0.f;
        if constexpr (KV8) {
          if (p.k_scales == nullptr) {
            x.k[t] *= fabsf(p.tensor_scale);
          } else {
            const int64_t idx = (int64_t)ids.v[t] * p.scale_pitch + kvh;
            const int tok = c * W::CT + t * 16;
            const bool there = tok < q.ctx && tok + 15 >= first_key(p, q);
            const float ks = load_uniform_f32(p.k_scales + idx), vs = load_uniform_f32(p.v_scales + idx);
            x.k[t] = there ? x.k[t] * ks : x.k[t];
            x.lv[t] = there && p.block_scales ? __builtin_amdgcn_logf(vs) : 0.f;
          }
        }
      }
      return x;
    };

    // columns
    const int map = MAPS == 2 ? i & 1 : 0, row = MAPS == 2 ? i >> 1 : i;
    const int j = row / G;
    const bool valid = row < q.n * G;
    const int head = kvh * G + (row - j * G);
    RowColumns<W> col;
    col.mul = 1.f;
    col.pos = attends_from(q, j);
    col.vis_hi = attends_from(q, 0);
    col.vis_lo = q.ctx - 1 - p.window;
    col.first = first_key(p, q);
    col.slope_log2 = (p.mask_flags & kMaskAlibi) && valid ? p.alibi_slopes[head] * kLog2e : 0.f;
    const char *qrow = p.query + (int64_t)(q.first + (valid ? j : 0)) * p.q_token_bytes + (valid ? head : 0) * p.q_head_bytes;
    u32x4 qv[W::KSTEPS];
#pragma unroll
    for (int c = 0; c < W::KSTEPS; ++c) {
      const int d0 = KV8 ? ((c >> 1) * 4 + r) * 16 + (c & 1) * 8 : (c * 4 + r) * 8;
      u32x4 z = {0u, 0u, 0u, 0u};
      const bool live = valid && (MAPS == 1 || (d0 >= D / 2) == (map == 1));
      qv[c] = live ? *reinterpret_cast<const u32x4 *>(qrow + d0 * 2) : z;
    }
    RowState st;
    st.m = st.mt = st.mv = st.mvt = -INFINITY;
    st.l = 0.f;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) wa.acc[dt] = f32x4{0.f, 0.f, 0.f, 0.f};

    if (ci < c_end) {
      typename W::Chunk R;
      typename W::Ids ids = wa.fetch_ids(table, ci, last_col);
      wa.issue_k(R, kvh, ci, ids);
      wa.issue_v(R, kvh, ci, ids);
      RowScales<TILES> sc = fetch_scales(ids, ci), nsc = sc;
      ids = wa.fetch_ids(table, ci + NW, last_col);
      if (KV8 && p.q_bf16) {
        float most = 0.f;
#pragma unroll
        for (int c = 0; c < W::KSTEPS; ++c) most = largest_of_bf16(qv[c], most);
        const uint32_t e = query_exponent(rows_max(most));
#pragma unroll
        for (int c = 0; c < W::KSTEPS; ++c) qv[c] = bf16_row_to_f16(qv[c], e);
        col.mul = bf16_row_scale(e);
      }
#pragma unroll
      for (int c = 0; c < W::KSTEPS; ++c)
#pragma unroll
        for (int k = 0; k < 4; ++k) wa.qB[c][k] = qv[c][k] ^ p.query_flip;
      while (ci + NW < c_end) {
        const int cn = ci + NW;
        const auto s = wa.qk(R);
        wa.issue_k(R, kvh, cn, ids);
        nsc = fetch_scales(ids, cn);
        const auto pb = row_soft<KV8, kTwo>(wa, st, col, R, s, sc, ci, q.ctx, p);
        wa.pv(R, pb.top);
        if constexpr (kTwo) wa.pv(R, pb.rest);
        wa.issue_v(R, kvh, cn, ids);
        ids = wa.fetch_ids(table, cn + NW, last_col);
        sc = nsc;
        ci = cn;
      }
      const auto s = wa.qk(R);
      const auto pb = row_soft<KV8, kTwo>(wa, st, col, R, s, sc, ci, q.ctx, p);
      wa.pv(R, pb.top);
      if constexpr (kTwo) wa.pv(R, pb.rest);
    }

    // Merge: sums and weights against the true maximum, then the wavefronts' states through LDS.  Wavefront w keeps the
    // slice [w * SL, (w + 1) * SL) of every lane's NR consecutive elements.
    {
      const float sink = MAPS == 1 && p.sinks != nullptr && valid && first == 0 && wave == 0 ? sink_log2(p, head) : -INFINITY;
      const float top = fmaxf(st.mt, sink), to = top == -INFINITY ? 0.f : top;
      const float from = KV8 && p.block_scales ? st.mv : st.m;
      const float f = from == -INFINITY ? 0.f : fast_exp2(from - to);
      st.l = rows_sum(st.l) * (st.m == -INFINITY ? 0.f : fast_exp2(st.m - to)) + fast_exp2(sink - to);
      float (*sm_acc)[NR][64] = reinterpret_cast<float (*)[NR][64]>(lds);
      float (*sm_m)[16] = reinterpret_cast<float (*)[16]>(lds + NW * NR * 64);
      float (*sm_l)[16] = reinterpret_cast<float (*)[16]>(lds + NW * NR * 64 + NW * 16);
      __syncthreads();  // (the piece before this one has been read)
      if (r == 0) {
        sm_m[wave][i] = top;
        sm_l[wave][i] = st.l;
      }
#pragma unroll
      for (int k = 0; k < NR; ++k) sm_acc[wave][k][lane] = wa.acc_at(k) * f;
      __syncthreads();
      float M = sm_m[0][i], L = 0.f, o[SL];
#pragma unroll
      for (int w = 1; w < NW; ++w) M = fmaxf(M, sm_m[w][i]);
      const float sub = M == -INFINITY ? 0.f : M;
#pragma unroll
      for (int k = 0; k < SL; ++k) o[k] = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float fw = fast_exp2(sm_m[w][i] - sub);
        L += fw * sm_l[w][i];
#pragma unroll
        for (int k = 0; k < SL; ++k) o[k] += fw * sm_acc[w][wave * SL + k][lane];
      }
      const float v_mul = !KV8 ? 1.f : p.block_scales ? 1.f : p.v_scales ? load_uniform_f32(p.v_scales + kvh) : p.tensor_scale;
      const int d0 = 4 * r * NDT + wave * SL;
      const bool whole = first == 0 && last == units;
      if (MAPS == 1 && whole) {
        if (valid) {
          const float inv = L == 0.f ? 0.f : v_mul / L;
          char *dst = p.out + (((int64_t)(q.first + j) * p.num_heads + head) * D + d0) * 2;
#pragma unroll
          for (int k = 0; k < SL; k += 2) *reinterpret_cast<uint32_t *>(dst + 2 * k) = pack_out(p, o[k] * inv, o[k + 1] * inv);
        }
      } else if (MAPS == 2 && whole) {
        // the maps of a row lie in neighbouring columns
        const float inv = L == 0.f ? 0.f : v_mul / L;
        const float lambda = p.lambdas[valid ? head : 0];
        float square = 0.f;
#pragma unroll
        for (int k = 0; k < SL; ++k) {
          const float mine = o[k] * inv;
          const float other = __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, mine), 0xB1, 0xF, 0xF, true));
          o[k] = mine - lambda * other;  // (of use in the columns of the first map)
          square += o[k] * o[k];
        }
        float mul = p.out_scale;
        if (p.norm_weight) {
          __syncthreads();  // the maxima have been read
          sm_m[wave][i] = rows_sum(square);
        }
        __syncthreads();
        if (p.norm_weight) mul = norm_factor(p, (sm_m[0][i] + sm_m[1][i] + sm_m[2][i] + sm_m[3][i]) / D);
        if (valid && map == 0) {
          char *dst = p.out + (((int64_t)(q.first + j) * p.num_heads + head) * D + d0) * 2;
          float w[SL];
#pragma unroll
          for (int k = 0; k < SL; ++k) w[k] = p.norm_weight ? mul * p.norm_weight[d0 + k] : mul;
#pragma unroll
          for (int k = 0; k < SL; k += 2) *reinterpret_cast<uint32_t *>(dst + 2 * k) = pack_out(p, o[k] * w[k], o[k + 1] * w[k + 1]);
        }
      } else {
        const int64_t slot = row_slot(p, kvh, seq, share);
        if (valid) {
          float *dst = p.row_o + (slot * kRowColumns + i) * D + d0;
#pragma unroll
          for (int k = 0; k < SL; k += 4)
            *reinterpret_cast<f32x4 *>(dst + k) = f32x4{o[k] * v_mul, o[k + 1] * v_mul, o[k + 2] * v_mul, o[k + 3] * v_mul};
        }
        if (wave == 0 && r == 0) {
          p.row_ml[slot * 2 * kRowColumns + i] = M;
          p.row_ml[slot * 2 * kRowColumns + kRowColumns + i] = L;
        }
      }
      if (first == 0 && kvh == 0 && threadIdx.x == 0 && !p.row_aligned)  // the shares that hold the sequence's pieces
        p.row_seqs[seq] = int2{share, (int)((((int64_t)before + units) * shares - 1) / total)};
    }
  } while (u < u_end);
}

// Joins the pieces of an item's rows.  Work-group (item, row): the pieces' maxima first, in LDS as factors; then the eight wavefronts
// sum every eighth piece each, with no load waiting for another.
template <int D, int MAPS>
__global__ void __launch_bounds__(512) ragged_rows_merge_kernel(const RaggedParams p) {
  constexpr int N = D / 64, NW = 8, kAhead = 4;
  __shared__ float factor[MAPS][kMaxRowGroups], ls[MAPS][kMaxRowGroups];
  __shared__ float sm[MAPS][NW][N][64], tops[MAPS][NW], sums[MAPS][NW];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int item = blockIdx.x, row = blockIdx.y;
  const int seq = item / p.num_kv_heads, kvh = item - seq * p.num_kv_heads;
  // (not set where the item has no keys; asked for with the lengths)
  const int first = load_uniform_i32(reinterpret_cast<const int32_t *>(p.row_seqs + seq));
  const int last = load_uniform_i32(reinterpret_cast<const int32_t *>(p.row_seqs + seq) + 1);
  const RaggedSeq q = ragged_seq_cut(p, ragged_seq_uniform(p.b, seq));
  if (row >= q.n * p.group || !in_rows_form<MAPS>(p, q)) return;
  const int j = row / p.group, head = kvh * p.group + (row - j * p.group);
  const int pieces = row_units<MAPS>(p, q) > 0 ? last - first + 1 : 0;
  if (pieces == 1) return;  // the rows kernel has stored the result
  const int64_t slot0 = row_slot(p, kvh, seq, first);
  float o[MAPS][N] = {};
  if (pieces > 0) {
    float early[MAPS][kAhead][N];  // the first pieces' values, asked for before the factors are known
#pragma unroll
    for (int m = 0; m < MAPS; ++m)
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int x = min(wave + u * NW, pieces - 1);
        const float *src = p.row_o + ((slot0 + x) * kRowColumns + row * MAPS + m) * D + lane * N;
#pragma unroll
        for (int k = 0; k < N; ++k) early[m][u][k] = src[k];
      }
#pragma unroll
    for (int m = 0; m < MAPS; ++m) {
      float top = -INFINITY;
      for (int x = threadIdx.x; x < pieces; x += 512) {
        const float *ml = p.row_ml + (slot0 + x) * 2 * kRowColumns + row * MAPS + m;
        const float pm = ml[0];
        factor[m][x] = pm;
        ls[m][x] = ml[kRowColumns];
        top = fmaxf(top, pm);
      }
      top = wave_max(top);
      if (lane == 0) tops[m][wave] = top;
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MAPS; ++m) {
      float top = tops[m][0];
#pragma unroll
      for (int w = 1; w < NW; ++w) top = fmaxf(top, tops[m][w]);
      const float sub = top == -INFINITY ? 0.f : top;
      float l = 0.f;
      for (int x = threadIdx.x; x < pieces; x += 512) {
        const float f = fast_exp2(factor[m][x] - sub);
        factor[m][x] = f;
        l += f * ls[m][x];
      }
      l = wave_sum(l);
      if (lane == 0) sums[m][wave] = l;
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MAPS; ++m) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const float f = wave + u * NW < pieces ? factor[m][wave + u * NW] : 0.f;
#pragma unroll
        for (int k = 0; k < N; ++k) o[m][k] += f == 0.f ? 0.f : f * early[m][u][k];
      }
#pragma unroll 8
      for (int x = wave + kAhead * NW; x < pieces; x += NW) {
        const float f = factor[m][x];
        const float *src = p.row_o + ((slot0 + x) * kRowColumns + row * MAPS + m) * D + lane * N;
#pragma unroll
        for (int k = 0; k < N; ++k) o[m][k] += f * src[k];
      }
#pragma unroll
      for (int k = 0; k < N; ++k) sm[m][wave][k][lane] = o[m][k];
    }
    __syncthreads();
  }
  if (wave != 0) return;
#pragma unroll
  for (int m = 0; m < MAPS; ++m) {
    float l = 0.f;
    if (pieces > 0) {
#pragma unroll
      for (int w = 0; w < NW; ++w) l += sums[m][w];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        o[m][k] = sm[m][0][k][lane];
#pragma unroll
        for (int w = 1; w < NW; ++w) o[m][k] += sm[m][w][k][lane];
      }
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
    for (int k = 0; k < N; ++k) o[m][k] *= inv;
  }
  if constexpr (MAPS == 2) {
    float x[N];
    differential_row<N>(p, head, lane, o[0], o[1], x);
    store_row<N>(p, q.first + j, head, lane, x);
  } else {
    store_row<N>(p, q.first + j, head, lane, o[0]);
  }
}

// The same for many items, of which few are in more than two or three pieces: a work-group for all rows of one, a wavefront
// for each row.  1024 items of 8 rows: 344 us with this kernel, 353 with the one above, whose 8192 work-groups find in the main that
// there is nothing to join; 152 items of up to 16 rows 133 and 130, a sequence in 64 pieces 44 and 20.
template <int D, int MAPS>
__global__ void __launch_bounds__(512) ragged_rows_join_kernel(const RaggedParams p) {
  constexpr int N = D / 64, NW = 8;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int seq = blockIdx.x / p.num_kv_heads, kvh = blockIdx.x - seq * p.num_kv_heads;
  // (not set where the sequence has no keys; asked for with the lengths)
  const int first = load_uniform_i32(reinterpret_cast<const int32_t *>(p.row_seqs + seq));
  const int last = load_uniform_i32(reinterpret_cast<const int32_t *>(p.row_seqs + seq) + 1);
  const RaggedSeq q = ragged_seq_cut(p, ragged_seq_uniform(p.b, seq));
  if (!in_rows_form<MAPS>(p, q)) return;
  const int pieces = row_units<MAPS>(p, q) > 0 ? last - first + 1 : 0;
  if (pieces == 1) return;  // the rows kernel has stored the result
  const int64_t slot0 = row_slot(p, kvh, seq, first);
  for (int row = wave; row < q.n * p.group; row += NW) {
    const int j = row / p.group, head = kvh * p.group + (row - j * p.group);
    float o[MAPS][N] = {};
#pragma unroll
    for (int m = 0; m < MAPS; ++m) {
      const float *ml = p.row_ml + slot0 * 2 * kRowColumns + row * MAPS + m;
      float top = -INFINITY;
      for (int x0 = 0; x0 < pieces; x0 += 64)
        top = fmaxf(top, wave_max(x0 + lane < pieces ? ml[(int64_t)(x0 + lane) * 2 * kRowColumns] : -INFINITY));
      const float sub = top == -INFINITY ? 0.f : top;
      float l = 0.f;
      for (int x0 = 0; x0 < pieces; x0 += 64) {
        const int here = min(64, pieces - x0);
        float f = 0.f;
        if (lane < here) {
          const float *at = ml + (int64_t)(x0 + lane) * 2 * kRowColumns;
          f = fast_exp2(at[0] - sub);
          l += f * at[kRowColumns];
        }
#pragma unroll 4
        for (int x = 0; x < here; ++x) {
          const float fx = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), x));
          const float *src = p.row_o + ((slot0 + x0 + x) * kRowColumns + row * MAPS + m) * D + lane * N;
#pragma unroll
          for (int k = 0; k < N; ++k) o[m][k] += fx * src[k];
        }
      }
      l = wave_sum(l);
      const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
      for (int k = 0; k < N; ++k) o[m][k] *= inv;
    }
    if constexpr (MAPS == 2) {
      float x[N];
      differential_row<N>(p, head, lane, o[0], o[1], x);
      store_row<N>(p, q.first + j, head, lane, x);
    } else {
      store_row<N>(p, q.first + j, head, lane, o[0]);
    }
  }
}

}  // namespace fa
