// Latent attention over the paged pool itself (absorbed form): every head's key is the cached row [c, r], every head's value its
// first part c.  Rows of the product are (new token, head) pairs, all heads of a token one after the other; they share one pass over
// the pool.
//
//   S^T[key, row] = [c, r] Q^T      MFMA 16x16x32, A = cached rows from LDS, B = queries, in registers for good
//   O^T[d, row]  += c^T P^T         MFMA 32x32x16, A = the same rows by transposing LDS reads, B = weights from LDS
//
// A work-group of eight wavefronts takes a tile of M rows (32, 64 or 128) and goes through 32 keys a step (bytes, M = 32: 64).  Cached rows go
// from memory to LDS by themselves (loads that write LDS), into a ring of steps.  A round is a matrix phase -- results of this step, scores of the
// next -- and a vector phase, the softmax:
//   M = 64, 128: four wavefronts, one on each SIMD, have the first half of the rows, the other four the second, one phase later, so that
//           one wavefront of a SIMD is in its matrix phase while the other is in its vector phase.  The second half loads, at the start of its
//           vector phase, where it has time (at the start of the matrix phase the same loads cost 350 of 1700 cycles).  A wavefront
//           has scores of 16 rows (M = 64: and half of the keys), and results of a half's rows for a quarter of the elements.
//   M = 32: all wavefronts are in the same phase; 16 rows and 16 keys (wavefronts without any load instead, where they can), an eighth of the
//           elements.
// Weights go through LDS, and so do the maxima of a row's keys where several wavefronts have them.
//
// Bytes of FP8 pools: M = 32 takes them from the ring as they are, and every wavefront decodes what it reads, half the LDS for
// a step of memory; M = 64 and 128 would decode each value four times in the time that the products take, so the wavefronts that load decode a
// step once, into a ring of 16-bit rows (64 heads, 13 sequences of 301 to 9000 keys, 2 to 6 tokens: a round of 32 keys and 128 rows
// 6000 -> 3900 cycles).
//
// Bound by memory where contexts are long (a round of 128 rows reads its 36 KiB at 5.0 TB/s over all compute units, of 32 rows of bytes at 6.0),
// by starts, ends and the join where they are short.  MI355X, both kernels: 128 heads over 64 sequences of 512 to 16384 keys 127 to 130 us (over
// machines), 16 heads over 128 FP8 sequences of 512 to 32768 keys 122 to 124 us, three users with 16 heads 15 us.
//
// Softmax against a reference m of each row that follows the maximum only where weights would pass 2^14 (kRefresh), and is set 2^6 below
// it then (kHeadroom); what there is of sums and results is multiplied then.  Weights carry the scale of their cached row (FP8 pools): w =
// 2^(score - m) scale, and so does the maximum; the sum does not.
// Weights are rounded to the queries' type, which the matrix cores take (their sum in 32 bits is that before the rounding): the result's error
// against 64 bits is 0.0020 to 0.0021 of its norm with bf16 and 0.00027 with fp16, where rounding the result alone makes 0.0017 and 0.0002.  A
// second part of each weight, as two maps have it, would double the products with the values.
//
// All tiles of the batch lie end to end on a line, each as long as its steps, and every work-group takes an equal share (LatentLine);
// pieces of cut tiles are joined by a second kernel.  Where sequences have several tiles, `team` of them lie side by side, and a share is
// that of as many work-groups, on one XCC: they go through the same keys at the same time, which come from memory once (64
// sequences of 512 to 16384 keys, 128 heads as two tiles of 64 rows: 352 MB fetched, and the pool has 346).
#pragma once

#include "latent_cache_kernel.h"
#include "ragged_tile_kernel.h"

namespace fa {

struct LatentJoin;
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
  int32_t groups;          // > 0: shares of the line, at most; 0: a work-group for each tile
  int32_t team;            // tiles side by side on the line
  float *part_o;           // pieces: [2 * (share * team + place in the team) + (0: its first, 1: a later one)][registers of its wavefronts]
  float *part_ml;          // [...][2][row]
  LatentJoin *joins;       // [share * team + place in the team]: the tile whose first cut is the end of the share
};

// A tile that is cut: its pieces are those of the shares first .. last (none: first > last).
struct LatentJoin {
  int32_t first, last, first_slot;  // first_slot: of the first share's piece; of the others 2 * (share * team + place in the team)
  int32_t first_token, row, rows;   // of the sequence; the tile's first row, the sequence's rows
};

// Keys of a step, what a tile costs apart from its steps, and the smallest share of the line (both in steps; 128 heads over 64 long sequences:
// kernel 108 us with kStart = 6, 103 with 12; three users with 16 heads: 14.4 us with kLeast = 8, 10.8 with 4).
template <bool KV8, int M>
struct LatentSteps {
  static constexpr int kKeys = KV8 && M == 32 ? 64 : 32, kStart = M == 128 ? 12 : KV8 && M == 32 ? 4 : 6, kLeast = KV8 && M == 32 ? 2 : 4;
};
constexpr float kNoReference = -1e30f;

// A sequence as its tiles see it.
struct LatentTiles {
  RaggedSeq q;
  int rows, tiles, teams, steps;  // steps of the last tile, at most what any tile has
  int64_t cost;                   // of a tile, or of those side by side
};
template <typename T>
__device__ __forceinline__ LatentTiles latent_tiles(const LatentParams &p, RaggedSeq q) {
  LatentTiles t;
  q.n = min(q.n, p.max_query_len);
  q.ctx = max(0, min(q.ctx, q.pos0 + q.n));
  t.q = q;
  t.rows = q.n * p.num_heads;
  t.tiles = (t.rows + T::kRows - 1) / T::kRows;
  t.teams = p.team == 1 ? t.tiles : (t.tiles + p.team - 1) / p.team;
  t.steps = (q.ctx + T::kKeys - 1) / T::kKeys;
  t.cost = t.steps + T::kStart;
  return t;
}
// Keys that the rows of a tile see: 0 .. latent_keys - 1.
template <typename T>
__device__ __forceinline__ int latent_keys(const LatentParams &p, const LatentTiles &t, int tile) {
  return max(0, attends_from(t.q, (min((tile + 1) * T::kRows, t.rows) - 1) / p.num_heads) + 1);
}

// Sum over the lanes below and with this one.
template <int CTRL, int ROWS>
__device__ __forceinline__ int64_t lanes_moved(int64_t v) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)((uint64_t)v >> 32), CTRL, ROWS, 0xf, false);
  return (int64_t)(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ int64_t wave_sums64(int64_t v) {
  v += lanes_moved<0x111, 0xf>(v);  // the lanes 1, 2, 4, 8 below, of 16
  v += lanes_moved<0x112, 0xf>(v);
  v += lanes_moved<0x114, 0xf>(v);
  v += lanes_moved<0x118, 0xf>(v);
  v += lanes_moved<0x142, 0xa>(v);  // lane 15 of the 16 before, to the second and the fourth 16
  v += lanes_moved<0x143, 0xc>(v);  // lane 31, to the last 32
  return v;
}
// Where share g of the line begins.  (Lengths on the line pass 32 bits, lengths of tiles do not.)
__host__ __device__ __forceinline__ int64_t latent_cut(int64_t total, int groups, int g) { return divide(total * g, groups); }
// The step that a cut `off` into a tile of `steps` steps lies before.
template <typename T>
__host__ __device__ __forceinline__ int latent_cut_step(int64_t off, int steps) {
  const int64_t step = off - T::kStart;
  return step <= 0 ? 0 : step < steps ? (int)step : steps;
}
// The shares that have steps of the tile of `steps` steps that begins at `start`, and whose first cut is the end of share g.
struct LatentShares {
  int first, last;
};
template <typename T>
__host__ __device__ __forceinline__ LatentShares latent_shares(int64_t total, int groups, int g, int64_t start, int steps) {
  const int64_t guess = divide((start + T::kStart + steps - 1) * groups, total) + 1;  // the last one, or one too many
  LatentShares s = {g, guess < groups ? (int)guess : groups - 1};
  while (latent_cut_step<T>(latent_cut(total, groups, s.first + 1) - start, steps) == 0) ++s.first;
  while (latent_cut(total, groups, s.last) - start - T::kStart >= steps) --s.last;
  return s;
}
template <typename T>
struct LatentPlace {
  int seq, team;  // team: which of the sequence's
  int64_t off;    // from its start
  LatentTiles t;
};
template <typename T>
struct LatentLine {
  int64_t total;
  int groups;
  RaggedSeq own;       // of the first 64 sequences: this lane's ...
  int64_t mine, upto;  // ... its length, and the sum up to it
  __device__ __forceinline__ LatentLine(const LatentParams &p, int lane) {
    own = ragged_seq_of_lane(p.b, min(lane, p.b.num_seqs - 1));
    mine = lane < p.b.num_seqs ? cost(p, own) : 0;
    upto = wave_sums64(mine);
    total = readlane64(upto, 63);
    if (p.b.num_seqs > 64) {
      int64_t more = 0;
      for (int s = 64 + lane; s < p.b.num_seqs; s += 64) more += cost(p, ragged_seq_of_lane(p.b, s));
      total += readlane64(wave_sums64(more), 63);
    }
    groups = (int)min((int64_t)p.groups, total / T::kLeast + (total > 0));
  }
  static __device__ __forceinline__ int64_t cost(const LatentParams &p, RaggedSeq q) {
    const LatentTiles t = latent_tiles<T>(p, q);
    return t.teams * t.cost;
  }
  __device__ __forceinline__ int64_t cut(int g) const { return latent_cut(total, groups, g); }
  // `at` < total
  __device__ __forceinline__ LatentPlace<T> find(const LatentParams &p, int64_t at, int lane) const {
    LatentPlace<T> r;
    int64_t before = 0, of_lane = mine, sum = upto;
    for (int base = 0;; base += 64) {
      if (base > 0) {
        of_lane = base + lane < p.b.num_seqs ? cost(p, ragged_seq_of_lane(p.b, base + lane)) : 0;
        sum = wave_sums64(of_lane);
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
    if (r.seq < 64) {
      r.t = latent_tiles<T>(p, RaggedSeq{__builtin_amdgcn_readlane(own.first, r.seq), __builtin_amdgcn_readlane(own.n, r.seq),
                                         __builtin_amdgcn_readlane(own.ctx, r.seq), __builtin_amdgcn_readlane(own.pos0, r.seq)});
    } else {
      r.t = latent_tiles<T>(p, ragged_seq_uniform(p.b, r.seq));
    }
    const int64_t in = at - before;
    r.team = __builtin_amdgcn_readfirstlane((int)divide(in, (int)r.t.cost));
    r.off = in - r.team * r.t.cost;
    return r;
  }
};

template <int L, typename OT, bool KV8, int M>
struct LatentAbsorbed : LatentSteps<KV8, M> {
  static constexpr int kRows = M, kKeys = LatentSteps<KV8, M>::kKeys;
  static constexpr bool kTurns = M >= 64;
  static constexpr bool kDecodes = KV8 && kTurns;               // rows of bytes are decoded once, into the ring
  static constexpr bool kBytes = KV8 && !kDecodes;              // ... or lie there as they are
  static constexpr int kRowElements = L + kLatentRope;
  static constexpr int kRowBytes = kRowElements * (kBytes ? 1 : 2);
  static constexpr int kStepBytes = kKeys * kRowBytes;
  static constexpr int kParts = kTurns ? 128 / M : kKeys / 16;  // of a step's keys, among wavefronts with the same rows
  static constexpr int kTiles = kKeys / 16 / kParts;            // of 16 keys, in a part
  static constexpr int kOwn = kBytes ? 16 : 8;                  // rows of a step that a wavefront loads
  static constexpr int kLoaders = kKeys / kOwn;                 // wavefronts that load, the last ones
  static constexpr int kPieces = kRowBytes / 16;                // of 16 bytes, of a row
  static constexpr int kLine = 64 / kOwn;                       // pieces of a row that one instruction loads
  static constexpr int kLoads = kDecodes ? (kRowElements + 127) / 128 : kPieces / kLine;  // instructions for the rows
  static constexpr int kInFlight = kLoads + KV8;                // ... and for their scales
  static constexpr int kRawStep = kDecodes ? kLoaders * kLoads * 1024 : 0;  // bytes of a step before they are decoded; two steps
  static constexpr int kOthers = 2 * kRawStep + M * kKeys * 2 + (kParts + 1) * M * 4 + M / 4 + (kDecodes ? 8 * kKeys * 4 : 0);  // LDS beside the ring
  static constexpr int kSlot = kStepBytes + (kBytes ? kKeys * 4 : 0);
  static constexpr int kRing = kDecodes ? 3 : (160 * 1024 - kOthers) / kSlot < 7 ? (160 * 1024 - kOthers) / kSlot : 7;
  static constexpr int kScaleSlots = kDecodes ? 8 : KV8 ? kRing : 0;
  static constexpr int kScales = kRing * kStepBytes;            // [slot][key]
  static constexpr int kRaw = kScales + kScaleSlots * kKeys * 4;
  static constexpr int kWeights = kRaw + 2 * kRawStep;          // [row][key] 16-bit
  static constexpr int kTops = kWeights + M * kKeys * 2;        // [part][row]: maxima
  static constexpr int kFactors = kTops + kParts * M * 4;       // [row]: what sums and results are multiplied with
  static constexpr int kFlags = kFactors + M * 4;               // [strip of 16 rows]: whether there are factors
  static constexpr int kLdsBytes = kFlags + M / 4;
  static constexpr int kBefore = kRing / 2;                     // steps in the ring before the queries' place
  static constexpr int kQueryRows = kParts == 1 ? 8 : 16;       // of a strip, in LDS at a time
  static constexpr int kSlices = kTurns ? 4 : 8;                // of the results' elements
  static constexpr int kResultTiles = M == 128 ? 2 : 1;         // of 32 rows
  static constexpr int DT = L / kSlices / 32, KS = kRowElements / 32;
  static_assert((kRing - kBefore) * kStepBytes >= M / 16 * kQueryRows * kRowElements * 2, "");
  static_assert(kLdsBytes <= 160 * 1024 && kRing >= (kDecodes ? 3 : 4) && (kRing - 1) * kInFlight < 64 && kPieces % kLine == 0, "");

  // The wavefronts' parts: a strip of 16 rows and a part of a step's keys for the scores, and whether a wavefront loads.
  static constexpr int strip_of(int wave) { return wave / kParts; }
  static constexpr int key_part_of(int wave) { return wave % kParts; }
  static constexpr bool loads(int wave) { return wave >= 8 - kLoaders; }
  // (M = 32: half of the wavefronts have no scores where there are 16 rows, or 32 keys a step)
  static constexpr bool has_scores(int strip, int rows) { return kTurns || strip * 16 < (M < rows ? M : rows); }
  // The first two wavefronts of a strip ask for its queries (one alone for all of them), and wait for whatever they have asked for, steps
  // of the ring among it.  Any other wavefront that loads waits for the first step by itself: it is read behind the next barrier.
  static constexpr bool asks_for_queries(bool scores, int key_part) { return kParts == 1 || (scores && key_part < 2); }
  static constexpr bool waits_for_first_step(bool scores, int key_part) { return !asks_for_queries(scores, key_part); }

  // Where 16-byte piece c of a row lies in a step's place in LDS: kOwn rows together, of each kLine pieces at a time, as the loads leave
  // them.  Which of the kLine goes by the row: then the 16 lanes of a read of 16 bytes that go together (0 .. 3, 12 .. 15 and 20 .. 27,
  // and the others) meet in no bank where they read two neighbouring pieces of 16 rows, nor do 32 lanes that read 4 rows of 64 bytes
  // (16-bit pools) or 8 rows of 32 bytes (bytes).
  static __device__ __forceinline__ int swizzle(int key) {
    return kBytes ? ((key >> 2) & 1) * 2 + ((key >> 3) & 1) : ((key >> 1) & 1) * 4 + (((key >> 2) ^ (key >> 3)) & 1) * 2 + ((key >> 3) & 1);
  }
  static __device__ __forceinline__ int piece_at(int key, int c) {
    return key / kOwn * kOwn * kRowBytes + c / kLine * 1024 + key % kOwn * kLine * 16 + ((c % kLine) ^ swizzle(key)) * 16;
  }
  // Where 16-byte piece c of a row of weights lies: 16 rows' same piece meets in no bank.
  static __device__ __forceinline__ int weights_at(int row, int c) {
    return kWeights + row * kKeys * 2 + (c ^ (kKeys == 32 ? (row >> 2) & 3 : (row >> 1) & 7)) * 16;
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
__device__ __forceinline__ void load_to_lds_16_from(uint32_t to, uint64_t address) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(address) : "memory");
}
// All but the last N loads of this wavefront have landed.
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// All but the last `steps` steps (MOST at most) of EACH loads.
template <int MOST, int EACH>
__device__ __forceinline__ void wait_steps(int steps) {
  if constexpr (MOST == 0) {
    wait_loads<0>();
  } else {
    if (steps >= MOST) wait_loads<MOST * EACH>();
    else wait_steps<MOST - 1, EACH>(steps);
  }
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
  constexpr int DT = T::DT, KS = T::KS, KT = T::kTiles, RT = T::kResultTiles;
  __shared__ __attribute__((aligned(16))) char lds[T::kLdsBytes];
  const uint32_t lds_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;

  const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31, quarter = lane >> 4, i16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // this wavefront's rows and keys of the scores, rows and elements of the results
  const int strip = T::strip_of(wave), key_part = T::key_part_of(wave), key0 = key_part * 16 * KT;
  const int result_row0 = T::kTurns ? (wave >> 2) * (M / 2) : 0, slice = wave % T::kSlices;
  const bool late = T::kTurns && wave >= 4, loads_here = T::loads(wave);
  const int loader = wave - (8 - T::kLoaders);  // which of those that load
  const int H = p.num_heads;

  // ---- this work-group's tiles ----
  LatentTiles t;
  int seq, team, from = 0, place = 0, part = blockIdx.x, end_seq, end_team, end_cut = 0x7fffffff;  // place: in the team
  if (p.groups > 0) {
    const LatentLine<T> line(p, lane);
    const int per = (line.groups + 7) >> 3, xcc = (int)blockIdx.x & 7, in_xcc = (int)blockIdx.x >> 3;  // work-groups go to the eight XCCs in turn:
    const int of_xcc = in_xcc / p.team, g = xcc * per + of_xcc;                                       // each gets an eighth of the line
    place = in_xcc % p.team, part = g * p.team + place;
    if (of_xcc >= per || g >= line.groups) {  // no share: nothing to join at its end
      const int idle = of_xcc >= per ? 8 * per + (of_xcc - per) * 8 + xcc : g;
      if (threadIdx.x == 0) p.joins[idle * p.team + place] = LatentJoin{1, 0, 0, 0, 0, 0};
      return;
    }
    const LatentPlace<T> at = line.find(p, line.cut(g), lane), to = line.find(p, line.cut(g + 1) - 1, lane);
    seq = at.seq, team = at.team, end_seq = to.seq, end_team = to.team;
    const LatentTiles &t1 = to.t;
    t = at.t;
    const int end_tile = to.team * p.team + place;
    const int end_steps = end_tile < t1.tiles ? (latent_keys<T>(p, t1, end_tile) + T::kKeys - 1) / T::kKeys : 0;
    from = latent_cut_step<T>(at.off, t.steps);
    if (to.off + 1 < t1.cost) end_cut = latent_cut_step<T>(to.off + 1, t1.steps);
    from = __builtin_amdgcn_readfirstlane(from), end_cut = __builtin_amdgcn_readfirstlane(end_cut);
    if (wave == 0) {  // what the join is told of the cut at this share's end
      LatentJoin join = {1, 0, 0, t1.q.first, end_tile * M, t1.rows};
      const int64_t start = line.cut(g + 1) - 1 - to.off;
      if (to.off + 1 < t1.cost && line.cut(g) <= start && end_steps > 0) {
        const LatentShares s = latent_shares<T>(line.total, line.groups, g, start, end_steps);
        if (s.first < s.last)
          join.first = s.first, join.last = s.last, join.first_slot = 2 * (s.first * p.team + place) + (s.first == g && line.cut(g) < start);
      }
      if (lane == 0) p.joins[part] = join;
    }
  } else {
    const RaggedPlace at = ragged_find(p.b.num_seqs, blockIdx.x, lane, [&](int s) { return latent_tiles<T>(p, ragged_seq_of_lane(p.b, s)).tiles; });
    seq = end_seq = __builtin_amdgcn_readfirstlane(at.seq);
    if (seq >= p.b.num_seqs) return;
    team = end_team = (int)blockIdx.x - __builtin_amdgcn_readfirstlane(at.before);
    t = latent_tiles<T>(p, ragged_seq_uniform(p.b, seq));
  }
  auto meet = [&]() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
  };

  // Bytes from a wavefront's first row of a step to the piece that this lane loads first; the next ones are kLine pieces on.
  // (Rows that are decoded: eight neighbouring pieces of bytes, then the last four, as the lanes come.)
  const uint32_t load_off = T::kDecodes ? (uint32_t)(lane >> 3) * p.token_bytes + (lane & 7) * 16
                                        : (uint32_t)(lane / T::kLine) * p.token_bytes + ((lane % T::kLine) ^ T::swizzle(lane / T::kLine + loader * T::kOwn)) * 16;
  // Where this lane reads: a cached row's piece for the scores, its transposed pieces for the results.  Two products or result tiles further on
  // are the next line.
  int row_at[2], value_at[4];
#pragma unroll
  for (int k = 0; k < 2; ++k) row_at[k] = T::kBytes ? T::piece_at(key0 + i16, 2 * k + (quarter >> 1)) + (quarter & 1) * 8 : T::piece_at(key0 + i16, 4 * k + quarter);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int key = 8 * half + (T::kBytes ? i16 >> 1 : (i16 >> 2) + (k >> 1) * 4);
    const int c = slice * (L / T::kSlices * (T::kBytes ? 1 : 2) / 16) + (T::kBytes ? (k & 1) * 2 + ((lane >> 4) & 1) : (k & 1) * 4 + ((lane >> 4) & 1) * 2 + ((i16 & 3) >> 1));
    value_at[k] = T::piece_at(key, c) + (i16 & 1) * 8;
  }
  float *tops = reinterpret_cast<float *>(lds + T::kTops), *factors = reinterpret_cast<float *>(lds + T::kFactors);
  int *flags = reinterpret_cast<int *>(lds + T::kFlags);

  bool first_piece = true;
  for (;; first_piece = false) {
    const RaggedSeq &q = t.q;
    const bool last_team = seq == end_seq && team == end_team;
    const int tile = team * p.team + place;
    const int keys = __builtin_amdgcn_readfirstlane(latent_keys<T>(p, t, tile));
    const int all_steps = (keys + T::kKeys - 1) / T::kKeys, until = last_team ? min(end_cut, all_steps) : all_steps;
    const bool whole = from == 0 && until == all_steps;
    if (tile < t.tiles && (whole || from < until)) {  // (a tile that sees no keys is whole: its rows get zeros)
      const int steps = until - from, row0 = tile * M;
      const bool scores_here = T::has_scores(strip, t.rows - row0);
      // this lane's row of the scores (rows past the end repeat the last one and are not stored)
      const int my_row = (strip * 16 + i16) & (M - 1), row = min(row0 + my_row, t.rows - 1);
      const int j = row / H, head = row - j * H, pos = attends_from(q, j);
      const int wave_lo = attends_from(q, min(row0 + strip * 16, t.rows - 1) / H);

      // This lane's row of queries.  It comes by way of LDS, where a strip of 16 rows has a place behind the steps that are asked for first:
      // rows may lie a power of two apart (heads outermost), and then 16 rows' same pieces, as the products take them, come from few
      // channels; a whole row at a time does not (128 heads of 64 tokens: a tile's start takes 17 000 cycles instead of 24 000).  Two wavefronts of a strip load
      // eight rows each; one alone loads and takes eight after the other.
      u32x4 qv[KS];
      const char *ql = p.query_latent + (int64_t)(q.first + j) * p.ql_token_bytes + head * p.ql_head_bytes;
      const char *qr = p.query_rope + (int64_t)(q.first + j) * p.qr_token_bytes + head * p.qr_head_bytes;
      auto load_queries = [&]() __attribute__((always_inline)) {
        constexpr int kPer = T::kQueryRows, kOfRow = L / 8, kRows1 = 512 / L;  // pieces of a row; rows to an instruction
        int lane_here = lane;  // (addresses are computed here, not kept over the steps)
        asm volatile("" : "+v"(lane_here));
        const int i16 = lane_here & 15, quarter = lane_here >> 4;
        const int place_at = T::kBefore * T::kStepBytes + strip * kPer * T::kRowElements * 2;
        const uint32_t to = (uint32_t)__builtin_amdgcn_readfirstlane(lds_at) + place_at;
        auto rows_to_lds = [&](int first, int at_row) __attribute__((always_inline)) {  // eight, to rows at_row .. of the place
#pragma unroll
          for (int i = 0; i < 8 / kRows1; ++i) {
            const int r = first + i * kRows1, piece = lane_here % kOfRow;
            uint64_t at = (uint64_t)readlane64((int64_t)(uintptr_t)ql, r);
            if (kRows1 == 2 && lane_here >= 32) at = (uint64_t)readlane64((int64_t)(uintptr_t)ql, r + 1);
            load_to_lds_16_from(to + (at_row + i * kRows1) * L * 2, at + ((piece ^ ((r + lane_here / kOfRow) & 7)) * 16));
          }
          const int r = first + (lane_here >> 3);
          load_to_lds_16_from(to + kPer * L * 2 + at_row * 128, (uint64_t)__shfl((long long)(uintptr_t)qr, r) + (((lane_here & 7) ^ (r & 7)) * 16));
        };
        auto from_lds = [&]() __attribute__((always_inline)) {
          const char *latent = lds + place_at + i16 % kPer * L * 2, *rope = lds + place_at + kPer * L * 2 + i16 % kPer * 128;
#pragma unroll
          for (int c = 0; c < KS; ++c)
            qv[c] = c < L / 32 ? *reinterpret_cast<const u32x4 *>(latent + ((4 * c + quarter) ^ (i16 & 7)) * 16)
                               : *reinterpret_cast<const u32x4 *>(rope + ((4 * (c - L / 32) + quarter) ^ (i16 & 7)) * 16);
        };
        if constexpr (kPer == 16) {
          if (T::asks_for_queries(scores_here, key_part)) {
            rows_to_lds(key_part * 8, key_part * 8);
            wait_loads<0>();
          }
          meet();
          if (scores_here) from_lds();
        } else {
          rows_to_lds(0, 0);
          wait_loads<0>();
          if (i16 < 8) from_lds();
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the next rows go to the same place
          rows_to_lds(8, 0);
          wait_loads<0>();
          if (i16 >= 8) from_lds();
        }
#pragma unroll
        for (int c = 0; c < KS; ++c)
#pragma unroll
          for (int k = 0; k < 4; ++k) qv[c][k] ^= p.query_flip;
      };
      float m = kNoReference, l = 0.f;
      f32x16 acc[RT][DT];
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[r][d][e] = 0.f;

      // ---- loads of a step: a wavefront has a quarter (an eighth) of its rows, which lie in one block ----
      const int32_t *table = p.b.block_tables + (int64_t)seq * p.b.max_blocks_per_seq;
      const int last_col = p.b.max_blocks_per_seq - 1, in_block = (1 << p.b.block_shift) - 1;
      auto id_of = [&](int n) { return load_uniform_i32(table + min(((from + n) * T::kKeys + loader * T::kOwn) >> p.b.block_shift, last_col)); };
      int32_t next_id = loads_here ? id_of(0) : 0;
      auto issue = [&](int n, int slot) __attribute__((always_inline)) {
        const uint32_t id = min((uint32_t)__builtin_amdgcn_readfirstlane(next_id), (uint32_t)p.b.max_block_id);
        const uint32_t r0 = (uint32_t)((from + n) * T::kKeys + loader * T::kOwn) & in_block;
        const char *base = uniform_address(p.cache + ((uint64_t)id * p.block_bytes + (uint64_t)r0 * p.token_bytes));
        const uint32_t lds0 = (uint32_t)__builtin_amdgcn_readfirstlane(lds_at);
        if constexpr (T::kDecodes) {
          const uint32_t to = lds0 + T::kRaw + (n & 1) * T::kRawStep + loader * T::kLoads * 1024;
#pragma unroll
          for (int i = 0; i < T::kLoads - 1; ++i) load_to_lds_16(to + i * 1024, load_off, base + i * 128);
          int last = lane;  // (computed here, not kept over the steps)
          asm volatile("" : "+v"(last));
          if (last < 32) load_to_lds_16(to + (T::kLoads - 1) * 1024, (uint32_t)(last >> 2) * p.token_bytes + (last & 3) * 16, base + (T::kLoads - 1) * 128);
        } else {
          const uint32_t to = lds0 + slot * T::kStepBytes + loader * T::kOwn * T::kRowBytes;
#pragma unroll
          for (int i = 0; i < T::kLoads; ++i) load_to_lds_16(to + i * 1024, load_off, base + i * T::kLine * 16);
        }
        if constexpr (KV8) {
          const char *scales = uniform_address(reinterpret_cast<const char *>(p.scales + (((uint64_t)id << p.b.block_shift) + r0)));
          if (lane < T::kOwn) load_to_lds_4(lds0 + T::kScales + ((T::kDecodes ? n & 7 : slot) * T::kKeys + loader * T::kOwn) * 4, lane * 4, scales);
        }
        next_id = id_of(n + 1);
      };
      // Rows of a step that no row of the tile sees may hold anything: zeros instead.  By the wavefront that has loaded them.
      auto clear_unseen = [&](int n, int slot) {
        const int k0 = (from + n) * T::kKeys + loader * T::kOwn;
#pragma unroll 1
        for (int r = min(max(keys - k0, 0), T::kOwn); r < T::kOwn; ++r) {
          char *dst = lds + slot * T::kStepBytes + loader * T::kOwn * T::kRowBytes + r * T::kLine * 16;
#pragma unroll 1
          for (int c = lane; c < T::kPieces; c += 64) *reinterpret_cast<u32x4 *>(dst + c / T::kLine * 1024 + c % T::kLine * 16) = u32x4{0u, 0u, 0u, 0u};
          if (KV8 && lane == 0) *reinterpret_cast<float *>(lds + T::kScales + ((T::kDecodes ? n & 7 : slot) * T::kKeys + loader * T::kOwn + r) * 4) = 0.f;
        }
      };

      // Rows of bytes of step n, which have landed, to their place in the ring; the step after next takes theirs.
      auto decode = [&](int n, int slot) __attribute__((always_inline)) {
        wait_steps<1, T::kInFlight>(min(steps - 1 - n, 1));
        int lane_here = lane;
        asm volatile("" : "+v"(lane_here));
        const char *src = lds + T::kRaw + (n & 1) * T::kRawStep + loader * T::kLoads * 1024 + lane_here * 16;
        char *dst = lds + slot * T::kStepBytes;
        const int key = loader * 8 + (lane_here >> 3), last_key = loader * 8 + ((lane_here >> 2) & 7);
        const int at = T::piece_at(key, 2 * (lane_here & 7)), last_at = T::piece_at(last_key, 2 * (lane_here & 3));
        u32x4 bytes[2] = {*reinterpret_cast<const u32x4 *>(src), *reinterpret_cast<const u32x4 *>(src + 1024)};
#pragma unroll
        for (int i = 0; i < T::kLoads; ++i) {
          __builtin_amdgcn_sched_barrier(0);
          const int to = (i < T::kLoads - 1 ? at : last_at) + i * 2048;
          if (i < T::kLoads - 1 || lane_here < 32) {
            *reinterpret_cast<u32x4 *>(dst + to) = decoded<OT>(u32x2{bytes[i & 1][0], bytes[i & 1][1]});
            *reinterpret_cast<u32x4 *>(dst + (to ^ 16)) = decoded<OT>(u32x2{bytes[i & 1][2], bytes[i & 1][3]});
          }
          if (i + 2 < T::kLoads) bytes[i & 1] = *reinterpret_cast<const u32x4 *>(src + (i + 2) * 1024);
        }
        if (n == steps - 1) clear_unseen(n, slot);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (n + 2 < steps) issue(n + 2, 0);
      };
      // Operands as LDS has them: 16-bit values, or bytes that are decoded before the product.
      using Raw = typename std::conditional<T::kBytes, u32x2, u32x4>::type;
      auto operand = [&](Raw a) {
        if constexpr (T::kBytes) return decoded<OT>(a);
        else return a;
      };
      auto row_operand = [&](const char *rows, int o) {  // product o: k-step o / KT of key tile o % KT
        const int c = o / KT;
        rows += o % KT * 16 * T::kRowBytes;
        if constexpr (T::kBytes) return *reinterpret_cast<const u32x2 *>(rows + row_at[c & 1] + (c >> 1) * 1024);
        else return *reinterpret_cast<const u32x4 *>(rows + row_at[c & 1] + (c >> 1) * 1024);
      };
      auto value_operand = [&](const char *rows, int ks, int d) {
        rows += 16 * ks * T::kRowBytes;
        if constexpr (T::kBytes) {
          return lds_read_transposed_bytes(rows + value_at[d & 1] + (d >> 1) * 1024);
        } else {
          const u32x2 a0 = lds_read_transposed(rows + value_at[d & 1] + (d >> 1) * 1024);
          const u32x2 a1 = lds_read_transposed(rows + value_at[2 + (d & 1)] + (d >> 1) * 1024);
          return u32x4{a0[0], a0[1], a1[0], a1[1]};
        }
      };

      // Scores of the step that softmax comes to next: element e of tile kt is key key0 + 16 kt + 4 quarter + e.
      f32x4 x[KT], s[KT];  // s: the rows' scales
      // ... times scale and log2(e), -inf where a key is not seen, and the largest of each row (in weights: with the rows' scales).
      auto scaled = [&](int n, int at) __attribute__((always_inline)) {
        const int t0 = (from + n) * T::kKeys + key0;
        float top = -INFINITY;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          if constexpr (KV8) s[kt] = *reinterpret_cast<const f32x4 *>(lds + T::kScales + ((T::kDecodes ? n & 7 : at) * T::kKeys + key0 + 16 * kt + 4 * quarter) * 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[kt][e] *= KV8 ? p.score_scale_log2 * s[kt][e] : p.score_scale_log2;
        }
        if (t0 + 16 * KT - 1 > wave_lo) {
          const int hi = pos - t0 - 4 * quarter;
#pragma unroll
          for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[kt][e] = 16 * kt + e > hi ? -INFINITY : x[kt][e];
        }
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int e = 0; e < 4; ++e) top = fmaxf(top, KV8 ? x[kt][e] + __builtin_amdgcn_logf(s[kt][e]) : x[kt][e]);
        return rows_max(top);
      };
      // The matrix phase: results of step n, then scores of step n + 1.  kAhead operands are on their way at any time; the order is held with
      // scheduling barriers, since left to itself the compiler asks for as many as there are and spills the rest.
      auto matrix_phase = [&](int n, int here, int next, auto with_scores, auto with_results) __attribute__((always_inline)) {
        constexpr bool kScores = decltype(with_scores)::value, kResults = decltype(with_results)::value;
        constexpr int kFirst = M == 128 ? 2 : 4, kAhead = M == 128 ? 4 : 6, kAll = KS * KT, kSteps = T::kKeys / 16, kFlagWords = M == 128 ? 4 : 2;
        constexpr int kValues = kSteps * DT, kLast = kFirst < kValues ? kFirst : kValues;
        const char *values = lds + here * T::kStepBytes, *rows = lds + next * T::kStepBytes;
        uint32_t moved[kFlagWords] = {};
        u32x4 b[kSteps][RT];
        auto weights = [&](int ks) __attribute__((always_inline)) {
#pragma unroll
          for (int r = 0; r < RT; ++r) b[ks][r] = *reinterpret_cast<const u32x4 *>(lds + T::weights_at(result_row0 + r * 32 + col, 2 * ks + half));
        };
        Raw a[kAhead];
        auto first_rows = [&](int upto) __attribute__((always_inline)) {  // score operands, asked for under the last results
#pragma unroll
          for (int o = 0; o < kAhead; ++o)
            if (o / 2 == upto) a[o] = row_operand(rows, o);
        };
        if constexpr (kResults) {
#pragma unroll
          for (int ks = 0; ks < (M == 128 ? 1 : kSteps); ++ks) weights(ks);
#pragma unroll
          for (int k = 0; k < kFlagWords; ++k) moved[k] = flags[result_row0 / 16 + k];
          Raw v[kFirst];
#pragma unroll
          for (int o = 0; o < kLast; ++o) v[o] = value_operand(values, o / DT, o % DT);
          uint32_t any = 0u;
#pragma unroll
          for (int k = 0; k < kFlagWords; ++k) any |= moved[k];
          if (__builtin_expect(__builtin_amdgcn_readfirstlane((int)any), 0)) {
#pragma unroll
            for (int r = 0; r < RT; ++r) {
              const bool is = col < 16 ? moved[2 * r] != 0u : moved[2 * r + 1] != 0u;
              const float f = is ? factors[result_row0 + r * 32 + col] : 1.f;
#pragma unroll
              for (int d = 0; d < DT; ++d) acc[r][d] *= f;
            }
          }
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int o = 0; o < kValues; ++o) {
            const u32x4 value = operand(v[o % kFirst]);
#pragma unroll
            for (int r = 0; r < RT; ++r) acc[r][o % DT] = mfma_32x32x16<OT>(value, b[o / DT][r], acc[r][o % DT]);
            if (M == 128 && o % DT == DT - 1 && o + 1 < kValues) weights(o / DT + 1);
            if (o + kFirst < kValues) v[o % kFirst] = value_operand(values, (o + kFirst) / DT, (o + kFirst) % DT);
            else if (kScores) first_rows(o + kLast - kValues);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        if constexpr (kScores) {
          f32x4 sum[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};  // two, for products that need not wait for each other
#pragma unroll
          for (int o = 0; o < kAhead; ++o)
            if (!kResults || o / 2 >= kLast) a[o] = row_operand(rows, o);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int o = 0; o < kAll; ++o) {
            sum[o & 1] = mfma_16x16x32<OT>(operand(a[o % kAhead]), qv[o / KT], sum[o & 1]);
            if (o + kAhead < kAll) a[o % kAhead] = row_operand(rows, o + kAhead);
            __builtin_amdgcn_sched_barrier(0);
          }
          if constexpr (KT == 1) x[0] = sum[0] + sum[1];
          else x[0] = sum[0], x[KT - 1] = sum[1];
        }
        if constexpr (kScores && T::kParts > 1) {  // for the other wavefronts that have keys of the row
          const float top = scaled(n + 1, next);
          if (quarter == 0) tops[key_part * M + my_row] = top;
        }
      };
      // The vector phase: weights of the scores, to LDS.
      auto softmax = [&](int n, int at) __attribute__((always_inline)) {
        float top;
        if constexpr (T::kParts == 1) {
          top = scaled(n, at);
        } else {
          top = tops[my_row];
#pragma unroll
          for (int k = 1; k < T::kParts; ++k) top = fmaxf(top, tops[k * M + my_row]);
        }
        int moved = 0;
        if (__builtin_expect(__any(top - m > kRefresh), 0)) {
          const float to = top - m > kRefresh ? top - kHeadroom : m, alpha = fast_exp2(m - to);
          l *= alpha;
          m = to;
          moved = 1;
          if (key_part == 0 && quarter == 0) factors[my_row] = alpha;
        }
        if (key_part == 0 && lane == 0) flags[strip] = moved;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          float w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            w[e] = fast_exp2(x[kt][e] - m);
            l += w[e];
            if constexpr (KV8) w[e] *= s[kt][e];
          }
          *reinterpret_cast<u32x2 *>(lds + T::weights_at(my_row, key0 / 8 + 2 * kt + (quarter >> 1)) + (quarter & 1) * 8) =
              u32x2{pack2<OT>(w[0], w[1]), pack2<OT>(w[2], w[3])};
        }
      };

      // ---- rounds: in round n the scores of step n + 1, the results of step n, and the softmax of step n + 1 ----
      if (!first_piece) meet();  // LDS of the piece before has been read
      if (threadIdx.x < M / 16) flags[threadIdx.x] = 0;  // (of rows that there are not)
      if (steps > 0) {
        constexpr int R = T::kRing;
        if (loads_here)
          for (int n = 0; n < min(T::kDecodes ? 2 : T::kBefore, steps); ++n) issue(n, n);
        load_queries();
        if constexpr (T::kDecodes) {
          if (loads_here) decode(0, 0);
        } else if (loads_here) {
          if (T::waits_for_first_step(scores_here, key_part)) wait_steps<T::kBefore - 1, T::kInFlight>(min(T::kBefore, steps) - 1);
          if (steps == 1) clear_unseen(0, 0);
        }
        meet();  // step 0 is there, and the queries' places are free
        if constexpr (T::kDecodes) {
          if (loads_here && steps > 1) decode(1, 1);
        } else if (loads_here) {
          for (int n = T::kBefore; n < min(R, steps); ++n) issue(n, n);
        }
        if (late) meet();
        int here = R - 1, next = 0;  // places in the ring of steps n, n + 1
        // Step n + 2 has landed, those after it are on their way.  (The late half does this before it asks for step n + R, others after.)
        auto land = [&](int n) __attribute__((always_inline)) {
          const int asked = min(max(n + (T::kTurns ? R - 1 : R), R - 1), steps - 1);
          wait_steps<R - 2, T::kInFlight>(asked - (n + 2));
          if (n + 2 == steps - 1) clear_unseen(n + 2, next + 1 == R ? 0 : next + 1);
        };
        auto round = [&](int n, auto with_results) __attribute__((always_inline)) {
          if (scores_here) matrix_phase(n, here, next, std::true_type{}, with_results);
          else matrix_phase(n, here, next, std::false_type{}, with_results);
          if (T::kTurns && !T::kDecodes && loads_here) land(n);
          meet();
          // step n has been read by all
          if (!T::kDecodes && loads_here && n >= 0 && n + R < steps) issue(n + R, here);
          if (scores_here) softmax(n + 1, next);
          if constexpr (T::kDecodes) {
            if (loads_here && n + R < steps) decode(n + R, here);
          }
          if (!T::kTurns && loads_here) land(n);
          meet();
          here = next, next = next + 1 == R ? 0 : next + 1;
        };
        round(-1, std::false_type{});
        for (int n = 0; n < steps - 1; ++n) round(n, std::true_type{});
        matrix_phase(steps - 1, here, next, std::false_type{}, std::true_type{});
        if (T::kTurns && !late) meet();
        meet();
      }

      // ---- results: element e of acc[r][d] is element slice L / slices + 32 d + 8 (e / 4) + 4 half + e % 4 of row result_row0 + 32 r + col ----
      float *stats = reinterpret_cast<float *>(lds + T::kWeights);  // references [M], then sums [M] of each part of the keys
      if (scores_here) {
        l = rows_sum(l);
        if (quarter == 0) {
          if (key_part == 0) stats[my_row] = m;
          stats[(1 + key_part) * M + my_row] = l;
        }
      }
      meet();
      auto sum_of = [&](int r) {
        float sum = stats[M + r];
#pragma unroll
        for (int k = 1; k < T::kParts; ++k) sum += stats[(1 + k) * M + r];
        return sum;
      };
      if (whole) {
        // by way of LDS, whole rows of the wavefront's elements at a time
        constexpr int kOfRow = DT * 4;  // 16-byte pieces, and lanes, of a row
        int lane_here = lane;           // (addresses are computed here, not kept over the steps)
        asm volatile("" : "+v"(lane_here));
        char *mine = lds + wave * 32 * DT * 64;
        const int row_in = lane_here / kOfRow, piece = lane_here % kOfRow;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const int of_tile = result_row0 + r * 32;
          const float sum = sum_of(of_tile + (lane_here & 31)), inv = sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              *reinterpret_cast<u32x2 *>(mine + (lane_here & 31) * (DT * 64) + (((4 * d + k) ^ ((lane_here & 31) & (kOfRow - 1))) * 16) + (lane_here >> 5) * 8) =
                  u32x2{pack2<OT>(acc[r][d][4 * k] * inv, acc[r][d][4 * k + 1] * inv), pack2<OT>(acc[r][d][4 * k + 2] * inv, acc[r][d][4 * k + 3] * inv)};
          __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
#pragma unroll
          for (int r0 = 0; r0 < 32; r0 += 64 / kOfRow) {
            const int of_wave = r0 + row_in, out_row = row0 + of_tile + of_wave;
            const u32x4 v = *reinterpret_cast<const u32x4 *>(mine + of_wave * (DT * 64) + ((piece ^ (of_wave & (kOfRow - 1))) * 16));
            const int token = out_row / H;
            if (out_row < t.rows)
              *reinterpret_cast<u32x4 *>(p.out + (int64_t)(q.first + token) * p.out_token_bytes + (out_row - token * H) * p.out_head_bytes + slice * (DT * 64) + piece * 16) = v;
          }
        }
      } else {
        // a piece: as it lies in the registers, 1 KiB at a time
        const int64_t slot = 2 * (int64_t)part + (first_piece ? 0 : 1);
        float *dst = p.part_o + (slot * 8 + wave) * (RT * DT * 1024) + lane * 4;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          if (row0 + result_row0 + r * 32 + col >= t.rows) continue;
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              *reinterpret_cast<f32x4 *>(dst + (r * DT + d) * 1024 + k * 256) = f32x4{acc[r][d][4 * k], acc[r][d][4 * k + 1], acc[r][d][4 * k + 2], acc[r][d][4 * k + 3]};
        }
        if (threadIdx.x < M) {
          p.part_ml[slot * 2 * M + threadIdx.x] = stats[threadIdx.x];
          p.part_ml[slot * 2 * M + M + threadIdx.x] = sum_of(threadIdx.x);
        }
      }
    }
    if (last_team) return;
    from = 0;
    if (++team >= t.teams) {
      team = 0;
      do {
        if (++seq >= p.b.num_seqs) return;  // (not while the arrays stay as they are)
        t = latent_tiles<T>(p, ragged_seq_uniform(p.b, seq));
      } while (t.teams == 0);
    }
  }
}

// Joins the pieces of cut tiles.  Work-group (x, y) has the x-th tile that is cut, if there are as many, and of it a product tile (32 rows, 32
// elements) of one wavefront.  Its four wavefronts go through the pieces in turn, four at a time so that their loads overlap, and meet in
// LDS.  (Sixteen wavefronts take as long, also where a tile has a hundred pieces.)
template <int L, typename OT, bool KV8, int M>
__global__ void __launch_bounds__(256) latent_absorbed_join_kernel(const LatentParams p) {
  using T = LatentAbsorbed<L, OT, KV8, M>;
  constexpr int DT = T::DT, kTiles = DT * T::kResultTiles;
  __shared__ float pieces[4][16][64], refs[4][2][64];
  const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  LatentJoin join = {1, 0, 0, 0, 0, 0};
  int found = -1;
  for (int base = 0, before = 0, all = p.groups * p.team; base < all && found < 0; base += 256) {
    LatentJoin its[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) its[k] = p.joins[min(base + k * 64 + lane, all - 1)];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool cut = base + k * 64 + lane < all && its[k].first <= its[k].last;
      const unsigned long long cuts = __ballot(cut), below = cuts & ((1ull << lane) - 1);
      const unsigned long long here = __ballot(cut && before + __popcll(below) == (int)blockIdx.x);
      if (found < 0 && here) {
        const int from = __builtin_ctzll(here);
        found = __builtin_amdgcn_readfirstlane(base + k * 64 + from);
        join = {__builtin_amdgcn_readlane(its[k].first, from),       __builtin_amdgcn_readlane(its[k].last, from),
                __builtin_amdgcn_readlane(its[k].first_slot, from),  __builtin_amdgcn_readlane(its[k].first_token, from),
                __builtin_amdgcn_readlane(its[k].row, from),         __builtin_amdgcn_readlane(its[k].rows, from)};
      }
      before += __popcll(cuts);
    }
  }
  if (found < 0) return;
  const int first = join.first, last = join.last, place = found % p.team;
  const int of_wave = blockIdx.y / kTiles, slice = of_wave % T::kSlices, d = blockIdx.y % DT;
  const int row0 = (T::kTurns ? (of_wave >> 2) * (M / 2) : 0) + blockIdx.y % kTiles / DT * 32;
  const int row = join.row + row0 + col;
  float m = kNoReference, l = 0.f;
  f32x16 acc;
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] = 0.f;
  struct Piece {
    float m, l;
    f32x4 o[4];
  };
  auto load = [&](int h) {
    Piece x = {kNoReference, 0.f, {}};
    if (row >= join.rows) return x;
    const int64_t slot = h == first ? join.first_slot : 2 * ((int64_t)h * p.team + place);
    const float *ml = p.part_ml + slot * 2 * M + row0 + col;
    const float *src = p.part_o + (slot * 8 * kTiles + blockIdx.y) * 1024 + lane * 4;
    x.m = ml[0], x.l = ml[M];
#pragma unroll
    for (int k = 0; k < 4; ++k) x.o[k] = *reinterpret_cast<const f32x4 *>(src + k * 256);
    return x;
  };
  auto add = [&](const Piece &x) {
    const float to = fmaxf(m, x.m), mine = fast_exp2(m - to), its = fast_exp2(x.m - to);
    l = l * mine + x.l * its;
    m = to;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = acc[e] * mine + x.o[e >> 2][e & 3] * its;
  };
  for (int h = first + wave; h <= last; h += 16) {
    Piece x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = load(min(h + 4 * k, last));
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (h + 4 * k <= last) add(x[k]);
  }
  refs[wave][0][lane] = m, refs[wave][1][lane] = l;
#pragma unroll
  for (int e = 0; e < 16; ++e) pieces[wave][e][lane] = acc[e];
  __syncthreads();
  // wavefront w finishes elements 8 w + 4 half + 0 .. 3
  if (row >= join.rows) return;
  float to = refs[0][0][lane], sum = 0.f, f[4];
#pragma unroll
  for (int w = 1; w < 4; ++w) to = fmaxf(to, refs[w][0][lane]);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    f[w] = fast_exp2(refs[w][0][lane] - to);
    sum += refs[w][1][lane] * f[w];
  }
  const int token = row / p.num_heads, head = row - token * p.num_heads;
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  char *dst = p.out + (int64_t)(join.first_token + token) * p.out_token_bytes + head * p.out_head_bytes + slice * (DT * 64) + d * 64 + wave * 16 + half * 8;
  float o[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    o[e] = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) o[e] += pieces[w][4 * wave + e][lane] * f[w];
    o[e] *= inv;
  }
  *reinterpret_cast<u32x2 *>(dst) = u32x2{pack2<OT>(o[0], o[1]), pack2<OT>(o[2], o[3])};
}

}  // namespace fa
