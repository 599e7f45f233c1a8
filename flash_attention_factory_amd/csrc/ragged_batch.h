// Ragged batches: a call brings the new tokens of all sequences one behind the other, query_start[s] .. query_start[s + 1] being
// those of sequence s, and context_lens[s] counts its keys with the new ones, so that its j-th new token of n sits at position
// context_lens[s] - n + j.  The arrays lie on the device; the host knows their sizes and bounds only.
#pragma once

#include "paged_attention_utils.h"

namespace fa {

struct RaggedBatch {
  const int32_t *query_start;   // [num_seqs + 1]
  const int32_t *context_lens;  // [num_seqs]
  const int32_t *block_tables;  // [num_seqs, max_blocks_per_seq]
  int32_t num_seqs;
  int32_t num_tokens;           // rows of the token arrays: what query_start says is cut to them
  int32_t max_blocks_per_seq;
  int32_t block_shift;          // log2(block_size)
  int32_t max_block_id;
};

// New tokens of a sequence: first row, how many, keys up to the last one's own, and the position of the first.  Rows that the token
// arrays do not have are not asked for, and keys that the block table cannot hold are not there; positions are those of
// the lengths as they are given, whatever has been cut.
struct RaggedSeq {
  int32_t first, n, ctx, pos0;
};
__device__ __forceinline__ RaggedSeq ragged_seq(const RaggedBatch &b, int s, int32_t start, int32_t end, int32_t len) {
  RaggedSeq q;
  q.first = min(max(start, 0), b.num_tokens);
  const int32_t all = max(end, q.first) - q.first;
  q.n = min(all, b.num_tokens - q.first);
  q.pos0 = max(len, 0) - all;
  q.ctx = max(0, min(q.pos0 + q.n, b.max_blocks_per_seq << b.block_shift));
  return q;
}
// for a sequence number that all lanes share (scalar loads) ...
__device__ __forceinline__ RaggedSeq ragged_seq_uniform(const RaggedBatch &b, int s) {
  return ragged_seq(b, s, load_uniform_i32(b.query_start + s), load_uniform_i32(b.query_start + s + 1),
                    load_uniform_i32(b.context_lens + s));
}
// ... and for one of each lane's own
__device__ __forceinline__ RaggedSeq ragged_seq_of_lane(const RaggedBatch &b, int s) {
  return ragged_seq(b, s, b.query_start[s], b.query_start[s + 1], b.context_lens[s]);
}

// Sum over the lanes below and with this one.
__device__ __forceinline__ int32_t wave_inclusive_scan(int32_t v, int lane) {
#pragma unroll
  for (int step = 1; step < 64; step <<= 1) {
    const int32_t other = __shfl_up(v, step);
    if (lane >= step) v += other;
  }
  return v;
}

// Which sequence holds item `u` of a list in which sequence s has count(s) items, and how many items lie before the
// sequence's own.  Every wavefront of a work-group looks for itself (no barrier): 64 sequences at a time, their counts summed
// across the lanes.  seq = num_seqs: the list has no item u; `before` is its length then.
struct RaggedPlace {
  int32_t seq, before;
};
template <typename Count>
__device__ __forceinline__ RaggedPlace ragged_find(int num_seqs, int32_t u, int lane, Count &&count) {
  int32_t carry = 0;
  for (int base = 0; base < num_seqs; base += 64) {
    const int s = base + lane;
    const int32_t mine = s < num_seqs ? count(s) : 0;
    const int32_t upto = wave_inclusive_scan(mine, lane);
    const unsigned long long beyond = __ballot(carry + upto > u);
    if (beyond) {
      const int at = __builtin_ctzll(beyond);
      const int32_t before = carry + __builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(mine, at);
      return {base + at, before};
    }
    carry += __builtin_amdgcn_readlane(upto, 63);
  }
  return {num_seqs, carry};
}

}  // namespace fa
