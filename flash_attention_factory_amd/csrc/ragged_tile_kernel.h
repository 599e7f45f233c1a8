// Ragged paged attention, tile form: many rows (new token, query head) per (sequence, kv head); bound by the matrix cores.
// Measured on an MI355X: 4096 new tokens after 12288 of a document, E4M3 pool (0.96 TFLOP), 0.95 to 1.0 ms, 1.0 PFLOP/s,
// where a large matrix product reaches 1.3; prompts with two maps (33 GFLOP) 65 us, 0.51 PFLOP/s; prompts next to
// running sequences (50 GFLOP) 111 us, of which the line of tiles takes 88 and its joins 16.  In the long case the matrix cores are busy
// for 43 % of the time and the vector units (exponentials, maxima, conversion of bytes) for 56 %, in the others for 20 to 23 % and 33
// to 39 %.
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
  // Key of a step that thread row `load_row` loads in a pass.  Where there are more thread rows than keys the surplus ones repeat the
  // others' (what they have loaded is not stored): a key beyond the step's 64 would lie, with blocks of more than 64, as
  // far beyond the end of its block.
  static __host__ __device__ constexpr int load_key(int pass, int load_row) {
    return kRowsPerPass > kTileKeys ? load_row & (kTileKeys - 1) : pass * kRowsPerPass + load_row;
  }

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

// ---- the line of tiles ----
// All tiles of the batch (sequence, kv head, tile of rows) laid end to end, each as long as it costs: about its keys, and
// kTileStart for what a tile costs apart from them.  Within a sequence the cost grows by the same amount from tile to
// tile (the causal rule), so sums and places have closed forms.  Work-group g takes the part from total * g / groups
// to total * (g + 1) / groups: equal shares, whatever the lengths are.  A cut within a tile becomes a cut between two steps.
// When this is done rather than one work-group per tile, longest first: ragged_plan, with both sides measured.
constexpr int kTileStart = 3 * kTileKeys;
constexpr int kLeastShare = 4 * kTileKeys;  // no shares smaller than that

struct TileCosts {
  int tiles;      // of one kv head
  int64_t first;  // cost of the first tile
  int64_t more;   // by which each costs more than the one before it
  __device__ __forceinline__ int64_t upto(int64_t t) const { return first * t + more * (t * (t - 1) / 2); }
  __device__ __forceinline__ int64_t of_head() const { return upto(tiles); }
};
template <int MAPS, int ROWS, typename Params>
__device__ __forceinline__ TileCosts tile_costs(const Params &p, RaggedSeq q) {
  TileCosts c;
  c.tiles = row_tiles<MAPS, ROWS>(p, q);
  q = ragged_seq_cut(p, q);
  const int tokens = ROWS / p.group + 1, all = min(max(q.pos0, 0), q.ctx);
  const int most = min(p.window, kNoWindow - tokens) + tokens;  // keys that a tile can see
  const int a = min(all + tokens, most), b = min(all + c.tiles * tokens, most);
  c.first = a + kTileStart;
  c.more = c.tiles > 1 ? (b - a) / (c.tiles - 1) : 0;
  return c;
}

__device__ __forceinline__ int64_t wave_inclusive_scan64(int64_t v, int lane) {
#pragma unroll
  for (int step = 1; step < 64; step <<= 1) {
    const int64_t other = __shfl_up(v, step);
    if (lane >= step) v += other;
  }
  return v;
}
__device__ __forceinline__ int64_t readlane64(int64_t v, int lane) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)v >> 32), lane);
  return (int64_t)(((uint64_t)hi << 32) | lo);
}

// A place on the line: the tile that lies there, and how far into it.
struct TilePlace {
  int seq, kvh, tile;
  int64_t off;  // cost units from the tile's start
};
// n / d for n and d below 2^53, without the 64-bit division's two hundred instructions.
template <typename Divisor>
__host__ __device__ __forceinline__ int64_t divide(int64_t n, Divisor d) {
  int64_t q = (int64_t)((double)n / (double)d);
  if (q * d > n) --q;
  if ((q + 1) * d <= n) ++q;
  return q;
}
template <int MAPS, int ROWS, typename Params = RaggedParams>
struct TileLine {
  int64_t total;
  int groups;
  int64_t mine, upto;  // of the first 64 sequences: this lane's, and the sum up to it
  __device__ __forceinline__ TileLine(const Params &p, int lane) {
    mine = costs(p, lane);
    upto = wave_inclusive_scan64(mine, lane);
    total = readlane64(upto, 63);
    if (p.b.num_seqs > 64) {
      int64_t more = 0;
      for (int s = 64 + lane; s < p.b.num_seqs; s += 64) more += costs(p, s);
      total += readlane64(wave_inclusive_scan64(more, lane), 63);
    }
    groups = (int)min((int64_t)p.tile_groups, total / kLeastShare + (total > 0));
  }
  static __device__ __forceinline__ int64_t costs(const Params &p, int s) {  // of all kv heads of sequence s
    return s < p.b.num_seqs ? tile_costs<MAPS, ROWS>(p, ragged_seq_of_lane(p.b, s)).of_head() * p.num_kv_heads : 0;
  }
  __device__ __forceinline__ int64_t cut(int g) const { return divide(total * g, groups); }
  // `at` < total
  __device__ __forceinline__ TilePlace find(const Params &p, int64_t at, int lane) const {
    TilePlace r;
    int64_t before = 0, of_lane = mine, sum = upto;
    for (int base = 0;; base += 64) {
      if (base > 0) {
        of_lane = costs(p, base + lane);
        sum = wave_inclusive_scan64(of_lane, lane);
      }
      const unsigned long long beyond = __ballot(before + sum > at);
      if (beyond || base + 64 >= p.b.num_seqs) {
        const int k = __builtin_ctzll(beyond | (1ull << 63));
        r.seq = __builtin_amdgcn_readfirstlane(base + k);
        before += readlane64(sum - of_lane, k);
        break;
      }
      before += readlane64(sum, 63);
    }
    const TileCosts c = tile_costs<MAPS, ROWS>(p, ragged_seq_uniform(p.b, r.seq));
    int64_t in = at - before;
    const int64_t head = c.of_head();
    int kvh = min((int)((float)in / (float)head), p.num_kv_heads - 1);
    while (kvh > 0 && in < head * kvh) --kvh;
    while (kvh + 1 < p.num_kv_heads && in >= head * (kvh + 1)) ++kvh;
    in -= head * kvh;
    // in >= first t + more t (t - 1) / 2: the root, then the whole number by comparison
    const float b = (float)c.first - 0.5f * (float)c.more;
    int t = c.more > 0 ? (int)((sqrtf(b * b + 2.0f * (float)c.more * (float)in) - b) / (float)c.more) : (int)((float)in / (float)c.first);
    t = min(max(t, 0), c.tiles - 1);
    while (t > 0 && in < c.upto(t)) --t;
    while (t + 1 < c.tiles && in >= c.upto(t + 1)) ++t;
    r.kvh = __builtin_amdgcn_readfirstlane(kvh);
    r.tile = __builtin_amdgcn_readfirstlane(t);
    r.off = in - c.upto(t);
    return r;
  }
};

// The steps of a tile: the first one, and how many (64 keys each).
struct TileSteps {
  int first, count;
};
template <int ROWS, typename Params>
__device__ __forceinline__ TileSteps tile_steps(const Params &p, const RaggedSeq &q, int tile) {
  const int row0 = tile * ROWS;
  const int pos_lo = attends_from(q, row0 / p.group), pos_hi = attends_from(q, (min(row0 + ROWS, q.n * p.group) - 1) / p.group);
  TileSteps s;
  s.first = max(0, pos_lo - p.window) / kTileKeys;
  s.count = pos_hi < 0 ? 0 : pos_hi / kTileKeys + 1 - s.first;
  return s;
}
// Where a cut `off` into a tile of cost `cost` falls between its steps.
__device__ __forceinline__ int cut_step(int64_t off, int64_t cost, int steps) {
  return min((int)((float)off * (float)steps / (float)cost), steps);
}

// The same number, as one that the compiler knows nothing of: what is worked out from it at a tile's end is not kept in registers from
// the tile's start, where it has been worked out before.  Two maps in a work-group for each tile have registers enough.
__device__ __forceinline__ int anew(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// What the wavefronts of a work-group have of a tile's rows: lane (half, col) holds elements d = 32 dt + 8 k + 4 half + e of row
// `strip * 32 + col` in acc[dt][4 k + e], against the maximum m with the sum l.  Normalises them, joins the maps, and stores the
// rows by way of LDS, 16 bytes per lane and whole rows at a time: eight bytes at a time into 32 rows cost more than four steps do.
// All wavefronts call it; LDS holds nothing else any more.
template <int D, int MAPS, int NW>
__device__ __forceinline__ void tile_finish(const RaggedParams &p, const RaggedSeq &q, int kvh, int row0, f32x16 (&acc)[D / 32], float l,
                                            char *lds, int lane) {
  constexpr int DT = D / 32, kRows = NW * 32 / MAPS;
  const int half = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int map = MAPS == 2 ? wave / (NW / 2) : 0, strip = MAPS == 2 ? wave % (NW / 2) : wave;
  const int all_rows = q.n * p.group, row = min(row0 + strip * 32 + col, all_rows - 1);
  const int j = row / p.group, head = kvh * p.group + (row - j * p.group);
  const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] *= inv;
  if constexpr (MAPS == 2) {  // second maps -> first maps (a lane's values at [value][lane] of its strip)
    float *through = reinterpret_cast<float *>(lds) + strip * DT * 16 * 64 + lane;
    if (map == 1) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) through[(dt * 16 + e) * 64] = acc[dt][e];
    }
    __syncthreads();
    if (map == 1) return;
    const float lambda = p.lambdas[head];
    float square = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        acc[dt][e] -= lambda * through[(dt * 16 + e) * 64];
        square += acc[dt][e] * acc[dt][e];
      }
    if (p.norm_weight) {
      f32x4 w[DT * 4];  // all asked for before the first is used
#pragma unroll
      for (int k = 0; k < DT * 4; ++k) w[k] = *reinterpret_cast<const f32x4 *>(p.norm_weight + 8 * k + 4 * half);
      const float mul = norm_factor(p, halves_sum(square) / D);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[dt][e] *= mul * w[dt * 4 + (e >> 2)][e & 3];
    } else {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) acc[dt] *= p.out_scale;
    }
  }
  // rows of D 16-bit values in the wavefront's own part of LDS, their 16-byte pieces swizzled by the row
  constexpr int kPer = D / 8;  // 16-byte pieces, and lanes, per row
  char *mine = lds + strip * 32 * D * 2 * MAPS;
  const auto put = [&](auto type) {
    using OutT = decltype(type);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        *reinterpret_cast<u32x2 *>(mine + col * (D * 2) + (((4 * dt + k) ^ (col & (kPer - 1))) * 16) + half * 8) =
            u32x2{pack2<OutT>(acc[dt][4 * k], acc[dt][4 * k + 1]), pack2<OutT>(acc[dt][4 * k + 2], acc[dt][4 * k + 3])};
  };
  if (p.q_bf16) put(BF16{});  // (asked once, not for every pair)
  else put(F16{});
  const int32_t out_row = (q.first + j) * p.num_heads + head;  // (num_tokens x num_heads fits 31 bits)
  const int left = all_rows - row0 - strip * 32;
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
#pragma unroll
  for (int r0 = 0; r0 < 32; r0 += 64 / kPer) {
    const int r = r0 + lane / kPer, c = lane & (kPer - 1);
    const int32_t to = __shfl(out_row, r);
    const u32x4 v = *reinterpret_cast<const u32x4 *>(mine + r * (D * 2) + ((c ^ (r & (kPer - 1))) * 16));
    if (r < left) *reinterpret_cast<u32x4 *>(p.out + (int64_t)to * (D * 2) + c * 16) = v;
  }
  static_assert(kRows * D * 2 * MAPS <= 4 * kTileKeys * D * 2 && (MAPS == 1 || kRows * D * 4 <= 4 * kTileKeys * D * 2), "it fits the buffers");
}

template <int D, typename OT, int KVF, int MAPS, int NW, bool EXT, bool LINE>
__global__ void __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(2))) ragged_tile_kernel(const RaggedParams p) {
  using T = RaggedTile<D, KVF, MAPS, NW>;
  constexpr bool KV8 = T::KV8;
  constexpr int KS = D / MAPS / 16;   // k-steps of the scores
  constexpr int DT = D / 32;          // d-tiles of the output
  constexpr bool kAnew = LINE || MAPS == 1;
  __shared__ __attribute__((aligned(16))) char lds[T::kLdsBytes];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5, col = lane & 31;
  const int map = MAPS == 2 ? wave / (NW / 2) : 0;
  const int strip = MAPS == 2 ? wave % (NW / 2) : wave;
  const int Hk = p.num_kv_heads, G = p.group;

  // This work-group's tiles: one, the last ones of a sequence first, since they see the most keys; or a share of the line.
  // Work-groups are handed to the eight XCCs in turn: each gets an eighth of the line, so that tiles of one kv head meet in
  // few L2 caches.
  int seq, kvh, tile, from = 0, g = 0, end_seq = 0, end_kvh = 0, end_tile = 0, end_cut = 0;
  bool first_piece = true;
  if constexpr (LINE) {
    const TileLine<MAPS, T::kRows> line(p, lane);
    const int per = (line.groups + 7) >> 3;
    g = ((int)blockIdx.x & 7) * per + ((int)blockIdx.x >> 3);
    if (((int)blockIdx.x >> 3) >= per || g >= line.groups) return;
    const TilePlace at = line.find(p, line.cut(g), lane), to = line.find(p, line.cut(g + 1) - 1, lane);
    seq = at.seq, kvh = at.kvh, tile = at.tile;
    end_seq = to.seq, end_kvh = to.kvh, end_tile = to.tile;
    const RaggedSeq q0 = ragged_seq_cut(p, ragged_seq_uniform(p.b, seq)), q1 = ragged_seq_cut(p, ragged_seq_uniform(p.b, end_seq));
    const TileCosts c0 = tile_costs<MAPS, T::kRows>(p, q0), c1 = tile_costs<MAPS, T::kRows>(p, q1);
    from = cut_step(at.off, c0.first + c0.more * tile, tile_steps<T::kRows>(p, q0, tile).count);
    const int64_t end_cost = c1.first + c1.more * end_tile;
    const int end_count = tile_steps<T::kRows>(p, q1, end_tile).count;
    end_cut = to.off + 1 == end_cost ? end_count : cut_step(to.off + 1, end_cost, end_count);
    from = __builtin_amdgcn_readfirstlane(from), end_cut = __builtin_amdgcn_readfirstlane(end_cut);
  } else {
    const int t = blockIdx.x / Hk;
    kvh = blockIdx.x - t * Hk;
    int before;
    if (p.b.num_seqs <= 64) {
      // Sequences with more keys first.  Each lane has one; its rank is the number of those before it, and what lies before it the
      // sum of their tiles.
      const RaggedSeq mine = lane < p.b.num_seqs ? ragged_seq_of_lane(p.b, lane) : RaggedSeq{0, 0, 0, 0};
      const int tiles = lane < p.b.num_seqs ? row_tiles<MAPS, T::kRows>(p, mine) : 0;
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
      const RaggedPlace at = ragged_find(p.b.num_seqs, t, lane,
                                         [&](int s) { return row_tiles<MAPS, T::kRows>(p, ragged_seq_of_lane(p.b, s)); });
      seq = __builtin_amdgcn_readfirstlane(at.seq);
      if (seq >= p.b.num_seqs) return;
      before = __builtin_amdgcn_readfirstlane(at.before);
    }
    tile = row_tiles<MAPS, T::kRows>(p, ragged_seq_uniform(p.b, seq)) - 1 - (t - before);
    end_seq = seq, end_kvh = kvh, end_tile = tile, end_cut = 0x7fffffff;
  }

  // Everything this work-group wrote to LDS is there, and nobody goes on before everybody is here.
  auto meet = [&]() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
  };

  for (;; first_piece = false) {
  const RaggedSeq q = ragged_seq_cut(p, ragged_seq_uniform(p.b, seq));
  const bool last_tile = !LINE || (seq == end_seq && kvh == end_kvh && tile == end_tile);
  const TileSteps of_tile = tile_steps<T::kRows>(p, q, tile);
  const int until = LINE && last_tile ? min(end_cut, of_tile.count) : of_tile.count;
  const bool whole = !LINE || (from == 0 && until == of_tile.count);
  if (whole || from < until) {  // (a tile that sees no keys is whole: its rows get zeros)
  const int all_rows = q.n * G, row0 = tile * T::kRows;
  const int step = of_tile.first + from, step_end = of_tile.first + until;

  // this lane's row (rows past the end repeat the last one and are not stored)
  const int my_row = row0 + strip * 32 + col;
  const int row = min(my_row, all_rows - 1);
  const int j = row / G, head = kvh * G + (row - j * G);
  const int pos = attends_from(q, j);
  const int wave_row = row0 + strip * 32;
  const bool wave_live = wave_row < all_rows;
  const int wave_lo = attends_from(q, min(wave_row, all_rows - 1) / G), wave_hi = attends_from(q, (min(wave_row + 32, all_rows) - 1) / G);

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
  const int steps = step_end - step;
  const int seen_lo = max(0, attends_from(q, row0 / G) - p.window);  // keys that some row of the tile sees
  const int seen_keys = attends_from(q, (min(row0 + T::kRows, all_rows) - 1) / G) + 1 - seen_lo;
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
    const int key = T::load_key(x, load_row);
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
    const int pass = KV8 ? w >> 1 : w, key = T::load_key(pass, load_row);
    const u32x4 o = lds_piece(kreg[pass], w);
    if (loads) *reinterpret_cast<u32x4 *>(lds + (n & 1) * T::kBufferBytes + T::k_at(key, KV8 ? 2 * piece + (w & 1) : piece)) = o;
  };
  auto write_v = [&](int n, int w) {
    const int pass = KV8 ? w >> 1 : w, key = T::load_key(pass, load_row);
    // what no row of the tile sees may be NaN
    if ((uint32_t)((step + n) * kTileKeys + key - seen_lo) >= (uint32_t)seen_keys) vreg[pass] = u32x4{0u, 0u, 0u, 0u};
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
  // block ids two steps ahead, the scales one step ahead, both left as they come until they are used.  Groups that no row sees
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
    const int key = (step + n) * kTileKeys + group_key;
    const float s = scaled && key < seen_lo + seen_keys && key + 15 >= seen_lo ? scale_raw : 1.f;
    const float log = p.block_scales ? __builtin_amdgcn_logf(s) : 0.f;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      sk[x] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, s), x));
      lv[x] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, log), 4 + x));
    }
  };

  // ---- the two phases of a step ----
  // (always inlined: a call would have everything that they work on, accumulators and all, go through memory)
  const float c_all = p.score_scale_log2 * q_mul * (KV8 && !scaled ? fabsf(p.tensor_scale) : 1.f);
  f32x16 x[2];   // scores of the step that softmax comes to next
  u32x4 pb[4];   // weights of the step before it, as the B operands of V^T P^T
  // (here the second part is products: prompts with two maps 64 us without, 80 with it.  bf16 takes it, with its 8 bits; fp16 does not,
  // and has an error of 0.00030 of the norm for it, where rounding the result alone makes 0.00021)
  constexpr bool kTwo = two_parts<KVF, MAPS>() && std::is_same<OT, BF16>::value;
  u32x4 rest[kTwo ? 4 : 1];  // what their rounding left
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
  constexpr int kScoreOps = 2 * KS, kValueOps = 4 * DT, kAhead = 4;
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
      if constexpr (kTwo) acc[dt] = mfma_32x32x16<OT>(a, rest[k], acc[dt]);
    }
  };
  // scores of step n + 1 and / or values of step n
  auto matrix_phase = [&](int n, auto with_scores, auto with_values, bool with_stage) __attribute__((always_inline)) {
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
  auto softmax = [&](int n) __attribute__((always_inline)) {
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
          // multiplied first: a factor may be 0 (keys of zeros have the least scale, queries of zeros the least exponent), and
          // -inf times 0 is NaN.  A select, since the pool may hold NaN there.
          x[t][e] = key > hi || key < lo ? -INFINITY : x[t][e] * cc[2 * t + (e >> 3)];
        }
#pragma unroll
      for (int k = 0; k < 4; ++k) cc[k] = 1.f;
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
      for (int w = 0; w < 4; ++w) {
        const float lo = x[k >> 1][(k & 1) * 8 + 2 * w], hi = x[k >> 1][(k & 1) * 8 + 2 * w + 1];
        pb[k][w] = pack2<OT>(lo, hi);
        if constexpr (kTwo) rest[k][w] = rest_of_pair<OT>(pb[k][w], lo, hi);
      }
    if constexpr (!blocks) {  // the sum of the weights as they are rounded: 16 instructions for 32 of them
      float part[2] = {0.f, 0.f};
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          part[w & 1] = add_pair<OT>(pb[k][w], part[w & 1]);
          if constexpr (kTwo) part[w & 1] = add_pair<OT>(rest[k][w], part[w & 1]);
        }
      l += part[0] + part[1];
    }
  };
  // ---- steps ----
  // Matrix phase of step n: scores of n + 1 and values of n, and between the products the thread's share of V of n + 1 and K of
  // n + 2 goes to LDS (what the next matrix phase reads) and the loads of the step after that are sent out.  Vector phase: softmax
  // of n + 1.  With eight wavefronts every SIMD has two: the second four run one phase behind the first, so that one is in its
  // matrix phase while the other is in its vector phase.
  if (LINE && !first_piece) meet();  // LDS of the piece before has been read
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
    auto vector_phase = [&](int n, auto with_softmax) __attribute__((always_inline)) {
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
    float sink = -INFINITY;
    if constexpr (MAPS == 1) {
      if (p.sinks != nullptr && from == 0) {
        const int row = min(row0 + strip * 32 + anew(col), all_rows - 1);
        sink = sink_log2(p, kvh * G + row % G);
        mt = fmaxf(mt, sink);
      }
    }
    const float to = mt == -INFINITY ? 0.f : mt;
    const float from = KV8 ? mv : m;
    const float v_mul = !KV8 || p.block_scales ? 1.f : p.v_scales ? load_uniform_f32(p.v_scales + kvh) : p.tensor_scale;
    const float f = (from == -INFINITY ? 0.f : fast_exp2(from - to)) * v_mul;
    l *= m == -INFINITY ? 0.f : fast_exp2(m - to);
    if constexpr (MAPS == 1) l += fast_exp2(sink - to);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt] *= f;
  }
  if (whole) {
    meet();  // nobody reads V any more
    tile_finish<D, MAPS, NW>(p, q, kvh, row0, acc, l, lds, kAnew ? anew(lane) : lane);
  } else {
    // a piece of a tile: as it lies in the registers, 1 KiB at a time (slots: see ragged_tile_merge_kernel)
    const int64_t slot = 2 * (int64_t)g + (first_piece ? 0 : 1);
    float *dst = p.tile_o + ((slot * NW + wave) * (DT * 4) * 64 + lane) * 4;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        *reinterpret_cast<f32x4 *>(dst + (dt * 4 + k) * 256) = f32x4{acc[dt][4 * k], acc[dt][4 * k + 1], acc[dt][4 * k + 2], acc[dt][4 * k + 3]};
    float *ml = p.tile_ml + (slot * NW + wave) * 128 + lane;
    ml[0] = mt;
    ml[64] = l;
  }
  }
  if (!LINE || last_tile) return;
  from = 0;
  if (++tile == row_tiles<MAPS, T::kRows>(p, q)) {
    tile = 0;
    if (++kvh == Hk) {
      kvh = 0;
      do {
        if (++seq >= p.b.num_seqs) return;  // (not while the arrays stay as they are)
      } while (row_tiles<MAPS, T::kRows>(p, ragged_seq_uniform(p.b, seq)) == 0);
    }
  }
  }
}

// Joins the pieces of a cut tile.  Work-group g looks at the cut between the shares of g and g + 1: if it is the first one within
// its tile, the pieces are those of g (its first, if its share begins with the tile, else its second one) and of the work-groups
// after it, whose first pieces they are.
template <int D, int MAPS, int NW>
__global__ void __launch_bounds__(NW * 64) ragged_tile_merge_kernel(const RaggedParams p) {
  constexpr int DT = D / 32, ROWS = NW * 32 / MAPS;
  __shared__ __attribute__((aligned(16))) char lds[4 * kTileKeys * D * 2];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const TileLine<MAPS, ROWS> line(p, lane);
  const int g = blockIdx.x;
  if (g + 1 >= line.groups) return;
  const int64_t at = line.cut(g + 1);
  const TilePlace place = line.find(p, at, lane);
  const int64_t start = at - place.off, before = line.cut(g);  // of the tile; of the share of g
  if (place.off == 0 || before > start) return;  // a cut between two tiles, or not the first one within its tile
  const RaggedSeq q = ragged_seq_cut(p, ragged_seq_uniform(p.b, place.seq));
  const TileCosts c = tile_costs<MAPS, ROWS>(p, q);
  const int64_t cost = c.first + c.more * place.tile;
  const int steps = tile_steps<ROWS>(p, q, place.tile).count;

  float m = -INFINITY, l = 0.f;
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
      const float pm = ml[0], to = fmaxf(m, pm), sub = to == -INFINITY ? 0.f : to;
      const float mine = fast_exp2(m - sub), its = fast_exp2(pm - sub);
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
  tile_finish<D, MAPS, NW>(p, q, place.kvh, place.tile * ROWS, acc, l, lds, lane);
}

}  // namespace fa
