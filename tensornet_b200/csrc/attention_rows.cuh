// Sequences, masks and scores as every attention kernel of this library sees them.
//
// Queries stand at the end of their keys: query i of a sequence with nq queries and nk keys stands at place i + nk - nq, or all of them,
// where they are newest, at nk - 1.  Key j is visible if j < nk and, where causal, j <= place or j < prefix: every mask is a limit per query, the number of keys it sees.
// Scores are kept in units of log2:  s = c q.k,  or cap tanh(scale q.k / cap) with a cap, less slope |place - j|.
#pragma once
#include <cuda_bf16.h>
#include <math_constants.h>
#include "attention.h"

namespace tn {
namespace attn {

constexpr float kLog2e = 1.4426950408889634f;

// Rows [first, first + n) of operand row b
struct Span {
  int b, first, n;
};
__device__ __forceinline__ int cut(int v, int lo, int hi) { return v < lo ? lo : (v > hi ? hi : v); }
__device__ __forceinline__ Span span_of(const AttnRows& r, int seq) {
  if (r.off == nullptr) return {seq, 0, r.len == nullptr ? r.T : cut(r.len[seq], 0, r.T)};
  const int lo = cut(r.off[seq], 0, r.T);
  return {0, lo, cut(r.off[seq + 1], lo, r.T) - lo};
}

// Tiles of `m` rows over all rows of an operand.  Padded: ceil(T / m) for each sequence, sequence after sequence, or, kByPlace, the first
// of every sequence, then the second: the work of a tile goes by its place where attention is causal, and blocks are started in the
// order of their work.  Packed: the rows in front of the first sequence, the sequences and the rows behind the last are segments 0 to
// B + 1 of [0, T); segment s has its first tile at number start(s) / m + s, which leaves room for ceil(n / m) tiles in each.
struct Tile {
  int seq;          // -1: rows that belong to no sequence
  Span rows;        // of the segment; padded: all T rows of the sequence
  int first;        // of the tile within the segment
  bool any;         // false: no such tile
};
__host__ __device__ __forceinline__ long long tile_count(const AttnRows& r, int B, int m) {
  return r.off == nullptr ? (long long)B * ((r.T + m - 1) / m) : (long long)r.T / m + B + 2;
}
// By a converged warp, all of whose lanes look at a segment each: three rounds of loads find one of 32768 sequences.
template <bool kByPlace>
__device__ __forceinline__ Tile tile_of(const AttnRows& r, int B, int m, int at) {
  if (r.off == nullptr) {
    const int per = kByPlace ? B : (r.T + m - 1) / m, slow = at / per, fast = at - slow * per, seq = kByPlace ? fast : slow;
    return {seq, {seq, 0, r.T}, (kByPlace ? slow : fast) * m, true};
  }
  auto start = [&](int s) { return s == 0 ? 0 : (s > B + 1 ? r.T : cut(r.off[s - 1], 0, r.T)); };
  int lo = 0, hi = B + 1;                                  // between them lies the last segment that starts at or before tile `at`
  while (lo < hi) {
    const int step = (hi - lo + 31) / 32, s = lo + ((int)(threadIdx.x & 31) + 1) * step;
    const bool before = s <= hi && start(s) / m + s <= at;
    lo += __popc(__ballot_sync(0xffffffffu, before)) * step;
    hi = min(hi, lo + step - 1);
  }
  const int s0 = start(lo), s1 = max(s0, start(lo + 1));
  const int first = (at - (s0 / m + lo)) * m;
  return {lo == 0 || lo == B + 1 ? -1 : lo - 1, {0, s0, s1 - s0}, first, first >= 0 && first < s1 - s0};
}

// keys that query i of a sequence sees
__device__ __forceinline__ int keys_seen(const AttnArgs& a, int seq, int i, int nq, int nk) {
  if (!a.causal) return nk;
  int lim = i + nk - nq + 1;
  if (a.prefix != nullptr) lim = max(lim, a.prefix[seq]);
  return cut(lim, 0, nk);
}

// the place of query i among the keys
__device__ __forceinline__ int place_of(const AttnArgs& a, int i, int nq, int nk) { return a.newest ? nk - 1 : i + nk - nq; }

// the first query of a sequence that sees key j
__device__ __forceinline__ int first_query(const AttnArgs& a, int seq, int j, int nq, int nk) {
  if (!a.causal || (a.prefix != nullptr && j < a.prefix[seq])) return 0;
  return max(0, j + nq - nk);
}

// of the sequences, as far as the host knows
__host__ __device__ __forceinline__ long long mean_length(const AttnRows& r, int B) { return r.off ? r.T / (B > 0 ? B : 1) : r.T; }

__device__ __forceinline__ long long flat_rows(const AttnRows& r, int B) { return r.off ? r.T : (long long)B * r.T; }

__device__ __forceinline__ const __nv_bfloat16* at(const AttnOperand& o, int b, long long t, int h) {
  return reinterpret_cast<const __nv_bfloat16*>(o.p) + b * o.sb + t * o.st + h * o.sh;
}
__device__ __forceinline__ __nv_bfloat16* at_out(const AttnOperand& o, int b, long long t, int h) {
  return reinterpret_cast<__nv_bfloat16*>(o.p) + b * o.sb + t * o.st + h * o.sh;
}

}  // namespace attn
}  // namespace tn
