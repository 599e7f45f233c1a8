// Latent attention over the paged pool itself (absorbed form): every head's key is the cached row [c, r], every head's value its
// first part c.  Rows of the product are (new token, head) pairs, all heads of a token one after the other; they share one pass over
// the pool.
//
//   S^T[key, row] = [c, r] Q^T      MFMA 16x16x32, A = cached rows from LDS, B = queries, in registers for good
//   O^T[d, row]  += c^T P^T         MFMA 32x32x16, A = the same rows by transposing LDS reads, B = weights from LDS
//
// A work-group of eight wavefronts takes a tile of M rows and goes through 32 keys a step.  Scores: 16 rows and 16 keys to a wavefront
// (M = 128: all 32; M = 32: four wavefronts have none).  Results: an eighth of the elements of all rows to a wavefront, so
// that a value read from LDS serves M / 32 products; weights go through LDS.  Cached rows go from memory to LDS by themselves (loads that
// write LDS), into a ring of steps, bytes of FP8 pools as they are: they are decoded on their way into the products.  One barrier a
// step: between two of them a wavefront makes its scores of the next step and its results of this one.
//
// Softmax against a reference m of each row that follows the maximum only where weights would pass 2^14 (kRefresh), and is set 2^6 below
// it then (kHeadroom).  A step in which some row's reference has to move is done again after its barrier (raise), by all wavefronts
// together.  Weights carry the scale of their row (FP8 pools): w = 2^(score - m) scale, and so does the maximum; the sum does not.
//
// All tiles of the batch lie end to end on a line, each as long as its steps, and every work-group takes an equal share (LatentLine);
// pieces of cut tiles are joined by a second kernel.
#pragma once

#include "latent_cache_kernel.h"
#include "ragged_tile_kernel.h"

namespace fa {

struct LatentParams {
  RaggedBatch b;
  const char *cache;
  const float *scales;
  uint32_t block_bytes, token_bytes;
  const char *query_latent, *query_rope;
  int64_t ql_token_bytes, ql_head_bytes, qr_token_bytes, qr_head_bytes;
  char *out;
  int64_t out_token_bytes, out_head_bytes;
  int32_t num_heads, max_query_len;
  float score_scale_log2;  // |scale| * log2(e)
  uint32_t query_flip;     // 0x80008000 for a negative scale
  int32_t groups;          // > 0: work-groups that share the line; 0: a work-group for each tile
  float *part_o;           // pieces: [2 * work-group + (0: its first, 1: a later one)][registers of its wavefronts]
  float *part_ml;          // [...][2][row]
};

constexpr int kLatentKeys = 32;       // keys of a step
constexpr int kLatentStart = 6;       // what a tile costs apart from its steps, in steps
constexpr int kLatentLeastShare = 8;  // no shares smaller than that, in steps
constexpr float kNoReference = -1e30f;

// A sequence as its tiles see it.
struct LatentTiles {
  RaggedSeq q;
  int rows, tiles, steps;  // steps of the last tile, at most what any tile has
  __device__ __forceinline__ int64_t cost() const { return steps + kLatentStart; }
  __device__ __forceinline__ int64_t all() const { return tiles * cost(); }
};
template <int M>
__device__ __forceinline__ LatentTiles latent_tiles(const LatentParams &p, RaggedSeq q) {
  LatentTiles t;
  q.n = min(q.n, p.max_query_len);
  q.ctx = max(0, min(q.ctx, q.pos0 + q.n));
  t.q = q;
  t.rows = q.n * p.num_heads;
  t.tiles = (t.rows + M - 1) / M;
  t.steps = (q.ctx + kLatentKeys - 1) / kLatentKeys;
  return t;
}
// Keys that the rows of a tile see: 0 .. latent_keys - 1.
template <int M>
__device__ __forceinline__ int latent_keys(const LatentParams &p, const LatentTiles &t, int tile) {
  return max(0, attends_from(t.q, (min(tile * M + M, t.rows) - 1) / p.num_heads) + 1);
}

struct LatentPlace {
  int seq, tile;
  int64_t off;  // from the tile's start
};
template <int M>
struct LatentLine {
  int64_t total;
  int groups;
  int64_t mine, upto;  // of the first 64 sequences: this lane's, and the sum up to it
  __device__ __forceinline__ LatentLine(const LatentParams &p, int lane) {
    mine = costs(p, lane);
    upto = wave_inclusive_scan64(mine, lane);
    total = readlane64(upto, 63);
    if (p.b.num_seqs > 64) {
      int64_t more = 0;
      for (int s = 64 + lane; s < p.b.num_seqs; s += 64) more += costs(p, s);
      total += readlane64(wave_inclusive_scan64(more, lane), 63);
    }
    groups = (int)min((int64_t)p.groups, total / kLatentLeastShare + (total > 0));
  }
  static __device__ __forceinline__ int64_t costs(const LatentParams &p, int s) {
    return s < p.b.num_seqs ? latent_tiles<M>(p, ragged_seq_of_lane(p.b, s)).all() : 0;
  }
  __device__ __forceinline__ int64_t cut(int g) const { return divide(total * g, groups); }
  // `at` < total
  __device__ __forceinline__ LatentPlace find(const LatentParams &p, int64_t at, int lane) const {
    LatentPlace r;
    int64_t before = 0, of_lane = mine, sum = upto;
    for (int base = 0;; base += 64) {
      if (base > 0) {
        of_lane = costs(p, base + lane);
        sum = wave_inclusive_scan64(of_lane, lane);
      }
      const unsigned long long beyond = __ballot(before + sum > at);
      if (beyond || base + 64 >= p.b.num_seqs) {
        const int k = __builtin_ctzll(beyond | (1ull << 63));
        r.seq = min(__builtin_amdgcn_readfirstlane(base + k), p.b.num_seqs - 1);
        before += readlane64(sum - of_lane, k);
        break;
      }
      before += readlane64(sum, 63);
    }
    const LatentTiles t = latent_tiles<M>(p, ragged_seq_uniform(p.b, r.seq));
    const int64_t in = at - before;
    r.tile = __builtin_amdgcn_readfirstlane((int)divide(in, (int)t.cost()));
    r.off = in - r.tile * t.cost();
    return r;
  }
};
// The step that a cut `off` into a tile of `steps` steps lies before.
__device__ __forceinline__ int latent_cut_step(int64_t off, int steps) { return min(max((int)off - kLatentStart, 0), steps); }

template <int L, typename OT, bool KV8, int M>
struct LatentAbsorbed {
  static constexpr int kRowElements = L + kLatentRope;
  static constexpr int kRowBytes = kRowElements * (KV8 ? 1 : 2);
  static constexpr int kStepBytes = kLatentKeys * kRowBytes;
  static constexpr int kRing = !KV8 && M == 128 && L == 512 ? 3 : 4;  // steps in LDS (4 of 36 KiB and more weights pass 160 KiB)
  static constexpr int kWeights = kRing * kStepBytes;                 // [2][M][32] 16-bit
  static constexpr int kScales = kWeights + 2 * M * 64;               // [ring][32]
  static constexpr int kTops = kScales + (KV8 ? kRing * 128 : 0);     // [2][M]: maxima of a step's halves, factors, sums
  static constexpr int kFlags = kTops + 2 * M * 4;                    // [2]: whether a reference has to move
  static constexpr int kLdsBytes = kFlags + 16;
  static constexpr int kPieces = kRowBytes / 16;                      // of 16 bytes, of a row
  static constexpr int kLoads = (4 * kPieces + 63) / 64;              // instructions for a wavefront's four rows
  static constexpr int kInFlight = kLoads + KV8;                      // ... and for their scales
  static constexpr int KT = M == 128 ? 2 : 1;                         // 16-key tiles of a wavefront's scores
  static constexpr int RT = M / 32, DT = L / 256, KS = kRowElements / 32;
  static_assert(kLdsBytes <= 160 * 1024, "");

  // Which 16-byte piece of a row lies at piece c of its place in LDS (and the other way round).  16 lanes that read one piece of 16
  // rows, and 32 that read 4 rows of 64 bytes (16-bit pools) or 8 rows of 32 bytes (bytes), meet in no bank.
  static __device__ __forceinline__ int swizzle(int key) {
    return KV8 ? ((key >> 2) & 1) * 2 + ((key >> 3) & 1) : ((key >> 1) & 1) * 4 + ((key >> 2) & 3);
  }
};

// 16 bytes for each lane from base + offset to LDS, `to` + 16 * lane; not waited for.  (m0 is the compiler's own scratch, set anew in front of
// every use.)
__device__ __forceinline__ void load_to_lds_16(uint32_t to, uint32_t offset, const char *base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(offset), "s"(base) : "memory");
}
__device__ __forceinline__ void load_to_lds_4(uint32_t to, uint32_t offset, const char *base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(to), "v"(offset), "s"(base) : "memory");
}
// All but the last N loads of this wavefront have landed.
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ const char *uniform_address(const char *p) {
  const uint64_t v = (uint64_t)(uintptr_t)p;
  return reinterpret_cast<const char *>(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32)) << 32) |
                                        (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v));
}
__device__ __forceinline__ u32x2 lds_read_transposed_bytes(const char *at) {
  typedef int i32x2 __attribute__((ext_vector_type(2)));
  typedef __attribute__((address_space(3))) i32x2 *lds_ptr;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_ptr)at));
}
// Eight E4M3 bytes as 16-bit values.
template <typename OT>
__device__ __forceinline__ u32x4 decoded(u32x2 bytes) {
  return u32x4{fp8_adjacent_pair<kKvE4M3, OT>(bytes[0], 0), fp8_adjacent_pair<kKvE4M3, OT>(bytes[0], 1),
               fp8_adjacent_pair<kKvE4M3, OT>(bytes[1], 0), fp8_adjacent_pair<kKvE4M3, OT>(bytes[1], 1)};
}

template <int L, typename OT, bool KV8, int M>
__global__ void __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) latent_absorbed_kernel(const LatentParams p) {
  using T = LatentAbsorbed<L, OT, KV8, M>;
  constexpr int RT = T::RT, DT = T::DT, KS = T::KS, KT = T::KT;
  __shared__ __attribute__((aligned(16))) char lds[T::kLdsBytes];
  const uint32_t lds_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;

  const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31, quarter = lane >> 4, i16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int strip = KT == 2 ? wave : wave >> 1, key0 = KT == 2 ? 0 : (wave & 1) * 16;  // this wavefront's rows and keys of the scores
  const bool scores_here = strip * 16 < M;
  const int H = p.num_heads;

  // ---- this work-group's tiles ----
  int seq, tile, from = 0, g = blockIdx.x, end_seq, end_tile, end_cut = 0x7fffffff;
  if (p.groups > 0) {
    const LatentLine<M> line(p, lane);
    const int per = (line.groups + 7) >> 3;  // work-groups go to the eight XCCs in turn: each gets an eighth of the line
    g = ((int)blockIdx.x & 7) * per + ((int)blockIdx.x >> 3);
    if (((int)blockIdx.x >> 3) >= per || g >= line.groups) return;
    const LatentPlace at = line.find(p, line.cut(g), lane), to = line.find(p, line.cut(g + 1) - 1, lane);
    seq = at.seq, tile = at.tile, end_seq = to.seq, end_tile = to.tile;
    const LatentTiles t0 = latent_tiles<M>(p, ragged_seq_uniform(p.b, seq)), t1 = latent_tiles<M>(p, ragged_seq_uniform(p.b, end_seq));
    from = latent_cut_step(at.off, (latent_keys<M>(p, t0, tile) + kLatentKeys - 1) / kLatentKeys);
    if (to.off + 1 < t1.cost()) end_cut = latent_cut_step(to.off + 1, (latent_keys<M>(p, t1, end_tile) + kLatentKeys - 1) / kLatentKeys);
    from = __builtin_amdgcn_readfirstlane(from), end_cut = __builtin_amdgcn_readfirstlane(end_cut);
  } else {
    const RaggedPlace at = ragged_find(p.b.num_seqs, blockIdx.x, lane, [&](int s) { return latent_tiles<M>(p, ragged_seq_of_lane(p.b, s)).tiles; });
    seq = end_seq = __builtin_amdgcn_readfirstlane(at.seq);
    if (seq >= p.b.num_seqs) return;
    tile = end_tile = (int)blockIdx.x - __builtin_amdgcn_readfirstlane(at.before);
  }
  auto meet = [&]() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
  };

  // Bytes from a wavefront's first row of a step to the piece that this lane loads, for each of its loads.
  uint32_t load_off[T::kLoads];
#pragma unroll
  for (int i = 0; i < T::kLoads; ++i) {
    const int slot = i * 64 + lane, r = min(slot / T::kPieces, 3), c = slot - slot / T::kPieces * T::kPieces;
    load_off[i] = (uint32_t)r * p.token_bytes + (c ^ T::swizzle(wave * 4 + r)) * 16;
  }
  const bool last_load = (T::kLoads - 1) * 64 + lane < 4 * T::kPieces;
  // Where this lane reads: a cached row's piece for the scores, its transposed pieces for the results, weights.  The swizzles are
  // exclusive-ors in the low bits of the pieces' numbers, so that some products or result tiles further on is an offset.
  constexpr int kRowBases = 2;
  int row_at[kRowBases], value_at[4];
#pragma unroll
  for (int k = 0; k < kRowBases; ++k) {
    const int key = key0 + i16;
    row_at[k] = key * T::kRowBytes + (KV8 ? ((2 * k + (quarter >> 1)) ^ T::swizzle(key)) * 16 + (quarter & 1) * 8 : ((4 * k + quarter) ^ T::swizzle(key)) * 16);
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (KV8) {
      const int key = 8 * half + (i16 >> 1), c = wave * (L / 128) + (k & 1) * 2 + ((lane >> 4) & 1);
      value_at[k] = key * T::kRowBytes + (c ^ T::swizzle(key)) * 16 + (i16 & 1) * 8;
    } else {
      const int key = 8 * half + (i16 >> 2) + (k >> 1) * 4, c = wave * (L / 64) + (k & 1) * 4 + ((lane >> 4) & 1) * 2 + ((i16 & 3) >> 1);
      value_at[k] = key * T::kRowBytes + (c ^ T::swizzle(key)) * 16 + (i16 & 1) * 8;
    }
  }
  float *tops = reinterpret_cast<float *>(lds + T::kTops);
  int *flags = reinterpret_cast<int *>(lds + T::kFlags);

  bool first_piece = true;
  for (;; first_piece = false) {
    const LatentTiles t = latent_tiles<M>(p, ragged_seq_uniform(p.b, seq));
    const RaggedSeq &q = t.q;
    const bool last_tile = seq == end_seq && tile == end_tile;
    const int keys = __builtin_amdgcn_readfirstlane(latent_keys<M>(p, t, tile));
    const int all_steps = (keys + kLatentKeys - 1) / kLatentKeys, until = last_tile ? min(end_cut, all_steps) : all_steps;
    const bool whole = from == 0 && until == all_steps;
    if (t.rows > 0 && (whole || from < until)) {  // (a tile that sees no keys is whole: its rows get zeros)
      const int steps = until - from, row0 = tile * M;
      // this lane's row of the scores (rows past the end repeat the last one and are not stored)
      const int my_row = (strip * 16 + i16) % M, row = min(row0 + my_row, t.rows - 1);
      const int j = row / H, head = row - j * H, pos = attends_from(q, j);
      const int wave_lo = attends_from(q, min(row0 + strip * 16, t.rows - 1) / H);

      u32x4 qv[KS];
      if (scores_here) {
        const char *ql = p.query_latent + (int64_t)(q.first + j) * p.ql_token_bytes + head * p.ql_head_bytes + quarter * 16;
        const char *qr = p.query_rope + (int64_t)(q.first + j) * p.qr_token_bytes + head * p.qr_head_bytes + quarter * 16;
#pragma unroll
        for (int c = 0; c < KS; ++c) {
          qv[c] = c < L / 32 ? *reinterpret_cast<const u32x4 *>(ql + c * 64) : *reinterpret_cast<const u32x4 *>(qr + (c - L / 32) * 64);
#pragma unroll
          for (int k = 0; k < 4; ++k) qv[c][k] ^= p.query_flip;
        }
      }
      float m = kNoReference, l = 0.f, part = 0.f;  // part: of the sum, by the step at hand
      f32x16 acc[DT][RT];
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[d][r][e] = 0.f;

      // ---- loads of a step: a wavefront has four of its rows, which lie in one block ----
      const int32_t *table = p.b.block_tables + (int64_t)seq * p.b.max_blocks_per_seq;
      const int last_col = p.b.max_blocks_per_seq - 1, in_block = (1 << p.b.block_shift) - 1;
      auto id_of = [&](int n) { return load_uniform_i32(table + min(((from + n) * kLatentKeys + wave * 4) >> p.b.block_shift, last_col)); };
      int32_t next_id = id_of(0);
      auto issue = [&](int n, int slot) __attribute__((always_inline)) {
        const uint32_t id = min((uint32_t)__builtin_amdgcn_readfirstlane(next_id), (uint32_t)p.b.max_block_id);
        const uint32_t r0 = (uint32_t)((from + n) * kLatentKeys + wave * 4) & in_block;
        const char *base = uniform_address(p.cache + ((uint64_t)id * p.block_bytes + (uint64_t)r0 * p.token_bytes));
        const uint32_t to = lds_at + slot * T::kStepBytes + wave * 4 * T::kRowBytes;
#pragma unroll
        for (int i = 0; i < T::kLoads; ++i) {
          if ((i + 1) * 64 <= 4 * T::kPieces || last_load) load_to_lds_16(__builtin_amdgcn_readfirstlane(to + i * 1024), load_off[i], base);
        }
        if constexpr (KV8) {
          const char *scales = uniform_address(reinterpret_cast<const char *>(p.scales + (((uint64_t)id << p.b.block_shift) + r0)));
          if (lane < 4) load_to_lds_4(__builtin_amdgcn_readfirstlane(lds_at + T::kScales + slot * 128 + wave * 16), lane * 4, scales);
        }
        next_id = id_of(n + 1);
      };
      // Rows of a step that no row of the tile sees may hold anything: zeros instead.  By the wavefront that has loaded them.
      auto clear_unseen = [&](int n, int slot) {
        const int k0 = (from + n) * kLatentKeys + wave * 4;
        for (int r = min(max(keys - k0, 0), 4); r < 4; ++r) {
          char *dst = lds + slot * T::kStepBytes + (wave * 4 + r) * T::kRowBytes;
          if (lane < T::kPieces) *reinterpret_cast<u32x4 *>(dst + lane * 16) = u32x4{0u, 0u, 0u, 0u};
          if (64 + lane < T::kPieces) *reinterpret_cast<u32x4 *>(dst + (64 + lane) * 16) = u32x4{0u, 0u, 0u, 0u};
          if (KV8 && lane == 0) *reinterpret_cast<float *>(lds + T::kScales + slot * 128 + (wave * 4 + r) * 4) = 0.f;
        }
      };

      // Operands as LDS has them: 16-bit values, or bytes that are decoded before the product.
      using Raw = typename std::conditional<KV8, u32x2, u32x4>::type;
      auto operand = [&](Raw a) {
        if constexpr (KV8) return decoded<OT>(a);
        else return a;
      };
      auto row_operand = [&](const char *rows, int c, int kt) {
        rows += kt * 16 * T::kRowBytes;
        if constexpr (KV8) return *reinterpret_cast<const u32x2 *>(rows + row_at[c & 1] + (c >> 1) * 64);
        else return *reinterpret_cast<const u32x4 *>(rows + row_at[c & 1] + (c >> 1) * 128);
      };
      auto value_operand = [&](const char *rows, int ks, int d) {
        rows += 16 * ks * T::kRowBytes;
        if constexpr (KV8) {
          return lds_read_transposed_bytes(rows + value_at[d & 1]);
        } else {
          const u32x2 a0 = lds_read_transposed(rows + value_at[d & 1]);
          const u32x2 a1 = lds_read_transposed(rows + value_at[2 + (d & 1)]);
          return u32x4{a0[0], a0[1], a1[0], a1[1]};
        }
      };

      f32x4 x[KT];  // scores of the step that is not summed yet: element e is key key0 + 16 kt + 4 quarter + e of the step
      auto scores = [&](int slot) __attribute__((always_inline)) {
        const char *rows = lds + slot * T::kStepBytes;
        // kAhead operands are on their way at any time; the order is held with scheduling barriers, since left to itself the compiler
        // asks for as many as there are and spills the rest
        constexpr int kAhead = 4, kAll = KS * KT;
        Raw a[kAhead];
#pragma unroll
        for (int o = 0; o < kAhead; ++o) a[o] = row_operand(rows, o / KT, o % KT);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int o = 0; o < kAll; ++o) {
          const int c = o / KT, kt = o % KT;
          x[kt] = mfma_16x16x32<OT>(operand(a[o % kAhead]), qv[c], c == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : x[kt]);
          if (o + kAhead < kAll) a[o % kAhead] = row_operand(rows, (o + kAhead) / KT, (o + kAhead) % KT);
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      float s[4 * KT];  // scales of the step's rows
      auto weights = [&](int n) __attribute__((always_inline)) {  // stores them, returns the largest
        float most = 0.f;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          float w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float v = fast_exp2(x[kt][e] - m);
            part = kt == 0 && e == 0 ? v : part + v;
            w[e] = KV8 ? v * s[4 * kt + e] : v;
          }
          most = max3(max3(most, w[0], w[1]), w[2], w[3]);
          const int at = key0 / 8 + 2 * kt + (quarter >> 1);
          *reinterpret_cast<u32x2 *>(lds + T::kWeights + ((n & 1) * M + my_row) * 64 + ((at ^ ((my_row >> 2) & 3)) * 16) + (quarter & 1) * 8) =
              u32x2{pack2<OT>(w[0], w[1]), pack2<OT>(w[2], w[3])};
        }
        return most;
      };
      auto softmax = [&](int n, int slot) __attribute__((always_inline)) {
        const int t0 = (from + n) * kLatentKeys + key0;
        l += part;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          f32x4 v = {1.f, 1.f, 1.f, 1.f};
          if constexpr (KV8) v = *reinterpret_cast<const f32x4 *>(lds + T::kScales + slot * 128 + (key0 + 16 * kt + 4 * quarter) * 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[4 * kt + e] = v[e];
            x[kt][e] *= KV8 ? p.score_scale_log2 * v[e] : p.score_scale_log2;
          }
        }
        if (t0 + 16 * KT - 1 > wave_lo) {
          const int hi = pos - t0 - 4 * quarter;
#pragma unroll
          for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[kt][e] = 16 * kt + e > hi ? -INFINITY : x[kt][e];
        }
        constexpr float kMost = 16384.f;  // 2^kRefresh
        if (__builtin_expect(__any(weights(n) > kMost), 0) && lane == 0) flags[n & 1] = 1;
      };
      // The references of step n move, where weights pass 2^kRefresh, and with them what there is of sums and results.
      auto raise = [&](int n) {
        if (scores_here) {
          float top = -INFINITY;
#pragma unroll
          for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int e = 0; e < 4; ++e) top = fmaxf(top, KV8 ? x[kt][e] + __builtin_amdgcn_logf(s[4 * kt + e]) : x[kt][e]);
          top = rows_max(top);
          if (quarter == 0) tops[(KT == 1 ? wave & 1 : 0) * M + my_row] = top;
        }
        meet();
        float alpha = 1.f;
        if (scores_here) {
          float top = tops[my_row];
          if (KT == 1) top = fmaxf(top, tops[M + my_row]);
          const float to = top > m + kRefresh ? top - kHeadroom : m;
          alpha = fast_exp2(m - to);
          l *= alpha;
          m = to;
          weights(n);
        }
        meet();
        if (scores_here && quarter == 0 && key0 == 0) tops[my_row] = alpha;
        if (threadIdx.x == 0) flags[n & 1] = 0;
        meet();
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const float f = tops[r * 32 + col];
#pragma unroll
          for (int d = 0; d < DT; ++d) acc[d][r] *= f;
        }
      };
      auto results = [&](int n, int slot) __attribute__((always_inline)) {
        const char *rows = lds + slot * T::kStepBytes;
        const char *from_weights = lds + T::kWeights + ((n & 1) * M + col) * 64;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          Raw a[DT];
          u32x4 b[RT];
#pragma unroll
          for (int d = 0; d < DT; ++d) a[d] = value_operand(rows, ks, d);
#pragma unroll
          for (int r = 0; r < RT; ++r)
            b[r] = *reinterpret_cast<const u32x4 *>(from_weights + r * 32 * 64 + (((2 * ks + half) ^ ((col >> 2) & 3)) * 16));
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            const u32x4 v = operand(a[d]);
#pragma unroll
            for (int r = 0; r < RT; ++r) acc[d][r] = mfma_32x32x16<OT>(v, b[r], acc[d][r]);
          }
        }
      };

      // ---- steps: in round n the scores of step n + 1 and the results of step n ----
      if (!first_piece) meet();  // LDS of the piece before has been read
      if (threadIdx.x < 2) flags[threadIdx.x] = 0;
      if (steps > 0) {
        constexpr int R = T::kRing;
        for (int n = 0; n < min(R - 2, steps); ++n) issue(n, n);
        if (steps > R - 3) wait_loads<(R - 3) * T::kInFlight>();
        else wait_loads<0>();
        if (steps == 1) clear_unseen(0, 0);
        meet();
        int here = 0, next = 1, far = R - 2;  // places in the ring of steps n, n + 1, n + R - 2
        auto land = [&](int n) {              // step n has landed, those after it are on their way
          if (n + R - 3 < steps) wait_loads<(R - 3) * T::kInFlight>();
          else wait_loads<0>();
          if (n == steps - 1) clear_unseen(n, next);
          meet();
        };
        if (R - 2 < steps) issue(R - 2, far);
        if (scores_here) {
          scores(0);
          softmax(0, 0);
        }
        land(1);
        for (int n = 0; n < steps - 1;) {
          if (__builtin_amdgcn_readfirstlane(flags[n & 1])) raise(n);
          do {
            far = far + 1 == R ? 0 : far + 1;
            if (n + R - 1 < steps) issue(n + R - 1, far);
            if (scores_here) scores(next);
            results(n, here);
            if (scores_here) softmax(n + 1, next);
            here = next, next = next + 1 == R ? 0 : next + 1;
            land(n + 2);
            ++n;
          } while (n < steps - 1 && !__builtin_amdgcn_readfirstlane(flags[n & 1]));
        }
        if (__builtin_amdgcn_readfirstlane(flags[(steps - 1) & 1])) raise(steps - 1);
        results(steps - 1, here);
        l += part;
        meet();
      }

      // ---- results: element e of acc[d][r] is element w L / 8 + 32 d + 8 (e / 4) + 4 half + e % 4 of row 32 r + col ----
      float *stats = reinterpret_cast<float *>(lds + T::kWeights);  // references [M], then sums [M] of each half of the keys
      if (scores_here) {
        l = rows_sum(l);
        if (quarter == 0) {
          if (key0 == 0) stats[my_row] = m;
          stats[(KT == 1 ? 1 + (wave & 1) : 1) * M + my_row] = l;
        }
      }
      meet();
      auto sum_of = [&](int r) { return KT == 1 ? stats[M + r] + stats[2 * M + r] : stats[M + r]; };
      if (whole) {
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const int out_row = row0 + r * 32 + col, stored = min(out_row, t.rows - 1), token = stored / H;
          const float sum = sum_of(r * 32 + col), inv = sum == 0.f ? 0.f : 1.0f / sum;
          char *dst = p.out + (int64_t)(q.first + token) * p.out_token_bytes + (stored - token * H) * p.out_head_bytes + wave * (L / 4) + half * 8;
          if (out_row < t.rows) {
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                *reinterpret_cast<u32x2 *>(dst + d * 64 + k * 16) = u32x2{pack2<OT>(acc[d][r][4 * k] * inv, acc[d][r][4 * k + 1] * inv),
                                                                          pack2<OT>(acc[d][r][4 * k + 2] * inv, acc[d][r][4 * k + 3] * inv)};
          }
        }
      } else {
        // a piece: as it lies in the registers, 1 KiB at a time
        const int64_t slot = 2 * (int64_t)g + (first_piece ? 0 : 1);
        float *dst = p.part_o + (slot * 8 + wave) * (DT * RT * 1024) + lane * 4;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              *reinterpret_cast<f32x4 *>(dst + (d * RT + r) * 1024 + k * 256) = f32x4{acc[d][r][4 * k], acc[d][r][4 * k + 1], acc[d][r][4 * k + 2], acc[d][r][4 * k + 3]};
        if (threadIdx.x < M) {
          p.part_ml[slot * 2 * M + threadIdx.x] = stats[threadIdx.x];
          p.part_ml[slot * 2 * M + M + threadIdx.x] = sum_of(threadIdx.x);
        }
      }
    }
    if (last_tile) return;
    from = 0;
    if (++tile >= t.tiles) {
      tile = 0;
      do {
        if (++seq >= p.b.num_seqs) return;  // (not while the arrays stay as they are)
      } while (latent_tiles<M>(p, ragged_seq_uniform(p.b, seq)).tiles == 0);
    }
  }
}

// Joins the pieces of a cut tile.  Work-groups (g, x) look at the cut between the shares of g and g + 1: if it is the first one within its
// tile, the pieces are those of g (its first, if its share begins with the tile, else its second one) and of the work-groups after
// it, whose first pieces they are.  x = d RT + r: one product tile of each wavefront.
template <int L, typename OT, bool KV8, int M>
__global__ void __launch_bounds__(512) latent_absorbed_join_kernel(const LatentParams p) {
  using T = LatentAbsorbed<L, OT, KV8, M>;
  constexpr int RT = T::RT, DT = T::DT;
  const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const LatentLine<M> line(p, lane);
  const int g = blockIdx.x, x = blockIdx.y, r = x % RT, d = x / RT;
  if (g + 1 >= line.groups) return;
  const int64_t at = line.cut(g + 1);
  const LatentPlace place = line.find(p, at, lane);
  const int64_t start = at - place.off, before = line.cut(g);  // of the tile; of the share of g
  if (place.off == 0 || before > start) return;  // a cut between two tiles, or not the first one within its tile
  const LatentTiles t = latent_tiles<M>(p, ragged_seq_uniform(p.b, place.seq));
  const int steps = (latent_keys<M>(p, t, place.tile) + kLatentKeys - 1) / kLatentKeys;
  const int64_t cost = t.cost();
  float m = kNoReference, l = 0.f;
  f32x16 acc;
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] = 0.f;
  int from = 0;
  for (int h = g;; ++h) {
    const int64_t share_end = h + 1 < line.groups ? line.cut(h + 1) : line.total;
    const bool last = share_end >= start + cost;
    const int until = __builtin_amdgcn_readfirstlane(last ? steps : latent_cut_step(share_end - start, steps));
    if (from == 0 && until == steps) return;  // one piece has it all: its work-group has stored the rows
    if (from < until) {
      const int64_t slot = 2 * (int64_t)h + (h == g && before < start ? 1 : 0);
      const float *ml = p.part_ml + slot * 2 * M + r * 32 + col;
      const float *src = p.part_o + ((slot * 8 + wave) * (DT * RT) + x) * 1024 + lane * 4;
      const float pm = ml[0], to = fmaxf(m, pm), mine = fast_exp2(m - to), its = fast_exp2(pm - to);
      l = l * mine + ml[M] * its;
      m = to;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const f32x4 o = *reinterpret_cast<const f32x4 *>(src + k * 256);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[4 * k + e] = acc[4 * k + e] * mine + o[e] * its;
      }
    }
    from = until;
    if (last) break;
  }
  const int row = place.tile * M + r * 32 + col;
  if (row >= t.rows) return;
  const int token = row / p.num_heads, head = row - token * p.num_heads;
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  char *dst = p.out + (int64_t)(t.q.first + token) * p.out_token_bytes + head * p.out_head_bytes + wave * (L / 4) + d * 64 + half * 8;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    *reinterpret_cast<u32x2 *>(dst + k * 16) =
        u32x2{pack2<OT>(acc[4 * k] * inv, acc[4 * k + 1] * inv), pack2<OT>(acc[4 * k + 2] * inv, acc[4 * k + 3] * inv)};
}

}  // namespace fa
