// Attention of a few queries against many keys, forward: up to 16 rows, a query head's query each, that share a key head.
//
// What bounds it is reading keys and values once.  A warp takes 16 or 32 keys at a time with a softmax and a ring of its own: one
// lane asks for tiles of keys and values by TMA, two or three steps ahead, so that a GPU's worth of warps has 28 MB on the way; products
// are mma.sync of 16 rows (at these rates far from what bounds it).  Tiles lie in rows of 128 bytes, swizzled, and are read
// 16 bytes at a time in the layout that the instruction wants, without conflicts:
//   * scores: the contraction may go over the columns in any order that both sides share.  A lane of group g = lane / 4, t = lane % 4
//     reads key spread(g) at column 8 t of 32: four words, the right operand of two products whose k are those columns.
//   * values: lane (g, t) reads keys t, t + 4, t + 8 and t + 12, which is where spread() has put the keys of its weights, at column
//     8 spread(g) of 64.  Words of two keys, interleaved by byte permutation, are the right operand of eight products; product i has
//     columns 8 spread(g) + i.
// spread() puts neighbouring groups four rows (or four pieces) apart, where the swizzle has the other half of the banks.
// Rows of 16 or 32 columns take pieces of 4 or 8 bytes of values in the same way.
// Measured: 512 histories of 20 to 2000 x 8 heads x 64 columns 89 us (5.1 TB/s), 2048 of 500 6.8 TB/s, 4 of 131072 x 2 key heads x 128
// 95 us with the kernel that joins the splits (5.6 TB/s; a sum over as many bytes takes 100 us).
// A sequence's keys are split over warps, blocks or both; what the blocks have of a row is brought to one reference and added by a
// second kernel, in a fixed order.
#include <cuda_bf16.h>
#include "attention_mma.cuh"

namespace tn {

namespace {

using namespace attn;

constexpr int kWarps = 4;
constexpr int kRowsM = 16;

struct FewPlan {
  int row_blocks;      // of 16 rows, of the queries of the heads that share a key head
  int splits;          // of a sequence's keys over blocks
  int chunk;           // keys of a split
  int per_unit;        // warps that share a split: 1 or kWarps
};

__device__ __forceinline__ int spread(int g) { return (g & 1) * 4 + (g >> 1); }

template <int kD>
struct FewShape : Pieces<kD> {
  static constexpr int keys = kD == 128 ? 16 : 32;                    // of a step
  static constexpr int chunks = kD == 128 ? 2 : 1;                    // of 64 columns
  static constexpr int chunk_bytes = keys * 128;
  static constexpr int stage_bytes = 2 * chunks * chunk_bytes;        // keys, then values: 8 KiB
  static constexpr int stages = kD == 128 ? 3 : 2;
  static constexpr int smem = kWarps * stages * stage_bytes + 1024;
};

struct FewMaps {
  CUtensorMap k, v;      // boxes of a step's keys
};

// part: [unit][split][16][kD] sums and [unit][split][16][2] references and sums of weights, where there are several splits
// kFar: the cap is above kCoarseCap
template <int kD, bool kFar>
__global__ void __launch_bounds__(32 * kWarps, kD == 128 ? 2 : 3)
attention_few_kernel(const __grid_constant__ FewMaps maps, const __grid_constant__ AttnArgs a, const FewPlan plan, float* __restrict__ part,
                     float* __restrict__ part_ml) {
  using S = FewShape<kD>;
  constexpr int kTilesN = S::keys / 8;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t s_full[kWarps][S::stages];
  __shared__ float s_m[kWarps][kRowsM], s_l[kWarps][kRowsM];
  __shared__ int s_abort_i;
  volatile int* s_abort = &s_abort_i;
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if (lane == 0) {
    for (int s = 0; s < S::stages; ++s) mbar_init(smem_u32(&s_full[warp][s]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    s_abort_i = 0;
  }
  __syncthreads();
  pdl_sync();
  const int R = a.H / a.G, rows = a.rq.T * R;
  const long long units = (long long)a.B * a.G * plan.row_blocks;
  const bool alone = plan.per_unit == 1;
  const long long unit = alone ? (long long)blockIdx.x * kWarps + warp : blockIdx.x;
  if (unit >= units) return;
  const int rb = (int)(unit % plan.row_blocks), kh = (int)(unit / plan.row_blocks % a.G), seq = (int)(unit / plan.row_blocks / a.G);
  const Span qs = span_of(a.rq, seq), ks = span_of(a.rk, seq);
  const int row0 = rb * kRowsM;
  // keys that the unit's last query sees; keys_seen grows with the query
  const int last = min((min(rows, row0 + kRowsM) - 1) / R, qs.n - 1);
  const int vis = row0 / R <= last ? keys_seen(a, seq, last, qs.n, ks.n) : 0;
  const int from = blockIdx.y * plan.chunk, to = min(vis, from + plan.chunk);
  const bool whole = vis <= plan.chunk;              // the first split has all there is to the unit's rows
  if (blockIdx.y > 0 && from >= to) return;          // the second kernel knows as much

  const uint32_t ring = ((smem_u32(smem_raw) + 1023u) & ~1023u) + warp * S::stages * S::stage_bytes;
  const uint8_t* ring_gen = smem_raw + (ring - smem_u32(smem_raw));
  const int stride = S::keys * plan.per_unit;
  const int j_first = from + (alone ? 0 : warp * S::keys);
  const int steps = j_first < to ? (to - j_first + stride - 1) / stride : 0;
  const bool lead = elect_one();
  auto ask = [&](int n) {
    const uint32_t bar = smem_u32(&s_full[warp][n % S::stages]), dst = ring + (n % S::stages) * S::stage_bytes;
    const int row = ks.first + j_first + n * stride;
    if (lead) {
      mbar_expect_tx(bar, S::stage_bytes);
#pragma unroll
      for (int c = 0; c < S::chunks; ++c) {
        tma_load_4d(dst + c * S::chunk_bytes, &maps.k, 64 * c, row, kh, ks.b, bar);
        tma_load_4d(dst + (S::chunks + c) * S::chunk_bytes, &maps.v, 64 * c, row, kh, ks.b, bar);
      }
    }
    __syncwarp();
  };
  for (int n = 0; n < S::stages && n < steps; ++n) ask(n);

  // row r of the unit: query (row0 + r) / R, query head kh * R + (row0 + r) % R
  int lim[2], place[2], least = vis;
  float slope2[2];
  uint32_t q[S::k_pieces * S::k_words][2];      // words of rows g and g + 8
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = row0 + g + 8 * e, i = r / R, h = kh * R + r % R;
    const bool there = r < rows && i < qs.n;
    lim[e] = there ? keys_seen(a, seq, i, qs.n, ks.n) : 0;
    if (there) least = min(least, lim[e]);
    place[e] = place_of(a, i, qs.n, ks.n);
    slope2[e] = there && a.slopes ? a.slopes[h] * kLog2e : 0.f;
#pragma unroll
    for (int p = 0; p < S::k_pieces; ++p) {
      const int d = (p * 4 + t) * 2 * S::k_words;
      uint32_t w[S::k_words] = {};
      if (there && d < a.D) load_words<S::k_words>(at(a.q, qs.b, i, h) + d, w);
#pragma unroll
      for (int i2 = 0; i2 < S::k_words; ++i2) q[p * S::k_words + i2][e] = w[i2];
    }
  }
  for (int o = 16; o > 0; o >>= 1) least = min(least, __shfl_xor_sync(0xffffffffu, least, o));

  float o[S::v_pieces * S::v_cols][4];
#pragma unroll
  for (int i = 0; i < S::v_pieces * S::v_cols; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m[2] = {kNone, kNone}, l[2] = {0.f, 0.f};
  const float cs = kFar ? a.scale / a.cap : a.cap > 0.f ? 2.f * kLog2e * a.scale / a.cap : a.scale * kLog2e;
  const float cap2 = a.cap * kLog2e;
  // where a lane reads: row spread(g) of eight for keys, rows t and t + 4 for values; the swizzle takes the row's number off the piece's
  const int k_row = spread(g), v_piece = kD >= 64 ? spread(g) : g;
  bool ok = true;
  for (int n = 0; n < steps; ++n) {
    const int j0 = j_first + n * stride;
    if (!mbar_wait_warp(smem_u32(&s_full[warp][n % S::stages]), (n / S::stages) & 1, s_abort)) { *s_abort = 1; ok = false; break; }
    const uint8_t* kt = ring_gen + (n % S::stages) * S::stage_bytes;
    const uint8_t* vt = kt + S::chunks * S::chunk_bytes;
    const bool masked = j0 + S::keys > min(least, to);
    float s[kTilesN][4];
#pragma unroll
    for (int c = 0; c < kTilesN; ++c) {
      s[c][0] = s[c][1] = s[c][2] = s[c][3] = 0.f;
#pragma unroll
      for (int p = 0; p < S::k_pieces; ++p) {
        uint32_t w[S::k_words];
        const int byte = (p * 4 + t) * 4 * S::k_words;          // of the row
        load_words<S::k_words>(kt + (byte >> 7) * S::chunk_bytes + (c * 8 + k_row) * 128 + ((byte & 127) ^ (k_row << 4)), w);
#pragma unroll
        for (int i = 0; i < S::k_words; i += 2) {
          const uint32_t aw[4] = {q[p * S::k_words + i][0], q[p * S::k_words + i][1], q[p * S::k_words + i + 1][0], q[p * S::k_words + i + 1][1]};
          mma16(s[c], aw, w[i], w[i + 1]);
        }
      }
    }
    // score e of product c: key j0 + 8 c + spread(2 t + (e & 1)) = j0 + 8 c + t + 4 (e & 1), row g + 8 (e >> 1)
    if (kFar)
#pragma unroll
      for (int c = 0; c < kTilesN; ++c)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float2 x = mul2(tanh_any<kCappedFar>(mul2(make_float2(s[c][2 * r], s[c][2 * r + 1]), both(cs))), both(cap2));
          s[c][2 * r] = x.x;
          s[c][2 * r + 1] = x.y;
        }
    float top[2] = {kNone, kNone};
#pragma unroll
    for (int c = 0; c < kTilesN; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = j0 + c * 8 + t + 4 * (e & 1), r = e >> 1;
        float x = kFar ? s[c][e] : s[c][e] * cs;
        if (!kFar && a.cap > 0.f) x = cap2 - __fdividef(2.f * cap2, 1.f + ex2(x));
        if (a.slopes != nullptr) x -= slope2[r] * fabsf((float)(place[r] - j));
        if (masked) x = j < min(lim[r], to) ? x : kNone;
        s[c][e] = x;
        top[r] = fmaxf(top[r], x);
      }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
    }
    if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float now = fmaxf(m[r], top[r]), by = now == kNone ? 1.f : ex2(m[r] - now);
        m[r] = now;
        l[r] *= by;
#pragma unroll
        for (int i = 0; i < S::v_pieces * S::v_cols; ++i) { o[i][2 * r] *= by; o[i][2 * r + 1] *= by; }
      }
    }
    const float ref[2] = {m[0] == kNone ? 0.f : m[0], m[1] == kNone ? 0.f : m[1]};
#pragma unroll
    for (int c = 0; c < kTilesN; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[c][e] = ex2(s[c][e] - ref[e >> 1]);
        l[e >> 1] += s[c][e];
      }
#pragma unroll
    for (int c = 0; c < S::keys / 16; ++c) {
      const uint32_t p[4] = {pack_bf16(s[2 * c][0], s[2 * c][1]), pack_bf16(s[2 * c][2], s[2 * c][3]), pack_bf16(s[2 * c + 1][0], s[2 * c + 1][1]),
                             pack_bf16(s[2 * c + 1][2], s[2 * c + 1][3])};
#pragma unroll
      for (int pc = 0; pc < S::v_pieces; ++pc) {
        uint32_t w[4][S::v_words];
        const int byte = v_piece * 4 * S::v_words;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = t + 4 * (e & 1);                      // of eight
          load_words<S::v_words>(vt + pc * S::chunk_bytes + (c * 16 + (e >> 1) * 8 + row) * 128 + (byte ^ (row << 4)), w[e]);
          if (masked && j0 + c * 16 + (e >> 1) * 8 + row >= to)      // what lies behind the sequence may be anything
#pragma unroll
            for (int i = 0; i < S::v_words; ++i) w[e][i] = 0u;
        }
        mma_values<S::v_words>(o + pc * S::v_cols, p, w);
      }
    }
    __syncwarp();
    if (n + S::stages < steps) ask(n + S::stages);
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    if (lim[r] <= 0) { l[r] = 0.f; m[r] = kNone; }
  }
  if (!ok) {
    if (lane == 0) set_status(a.status, kMbarTimeout, 43, (int)blockIdx.x);
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);        // copies in flight land
  }

  // Lane (g, t) has of row g + 8 r the columns (8 p + piece(2 t + f)) v_cols + i, f < 2, i < v_cols: value o[p v_cols + i][2 r + f],
  // where piece() is spread() as for the values read.
  const long long q_rows = (long long)a.B * a.rq.T;
  auto column = [&](int p, int f) { return (p * 8 + (kD >= 64 ? t + 4 * f : 2 * t + f)) * S::v_cols; };
  if (alone) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = row0 + g + 8 * r;
      if (row >= rows) continue;
      if (!whole) {
        const long long at_part = (unit * plan.splits + blockIdx.y) * kRowsM + g + 8 * r;
#pragma unroll
        for (int p = 0; p < S::v_pieces; ++p)
#pragma unroll
          for (int f = 0; f < 2; ++f)
#pragma unroll
            for (int k = 0; k < S::v_cols; k += 2)
              *reinterpret_cast<float2*>(part + at_part * kD + column(p, f) + k) = make_float2(o[p * S::v_cols + k][2 * r + f], o[p * S::v_cols + k + 1][2 * r + f]);
        if (t == 0) *reinterpret_cast<float2*>(part_ml + 2 * at_part) = make_float2(m[r], l[r]);
        continue;
      }
      const int i = row / R, h = kh * R + row % R;
      const float w = l[r] > 0.f ? 1.f / l[r] : 0.f;
      __nv_bfloat16* out = at_out(a.o, seq, i, h);
#pragma unroll
      for (int p = 0; p < S::v_pieces; ++p)
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          const int d = column(p, f);
          if (d >= a.D) continue;
          uint32_t v[S::v_words], rest[S::v_words];
#pragma unroll
          for (int k = 0; k < S::v_words; ++k) {
            const float x = o[p * S::v_cols + 2 * k][2 * r + f] * w, y = o[p * S::v_cols + 2 * k + 1][2 * r + f] * w;
            v[k] = pack_bf16(x, y);
            rest[k] = rest_of(x, y, v[k]);
          }
          store_words<S::v_words>(out + d, v);
          if (a.rest.p != nullptr) store_words<S::v_words>(at_out(a.rest, seq, i, h) + d, rest);
        }
      if (a.lse != nullptr && t == 0) a.lse[h * q_rows + (long long)seq * a.rq.T + i] = l[r] > 0.f ? m[r] + log2f(l[r]) : CUDART_INF_F;
    }
    return;
  }
  if (t == 0)
#pragma unroll
    for (int r = 0; r < 2; ++r) { s_m[warp][g + 8 * r] = m[r]; s_l[warp][g + 8 * r] = l[r]; }
  __syncthreads();              // and every warp is through with its ring
  float* s_o = reinterpret_cast<float*>(smem_raw);                    // [warp][16][kD + 4]
  constexpr int kPitch = kD + 4;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    if (row0 + g + 8 * r >= rows) continue;
    float all = kNone;
    for (int w = 0; w < kWarps; ++w) all = fmaxf(all, s_m[w][g + 8 * r]);
    const float by = m[r] == kNone ? 0.f : ex2(m[r] - all);
#pragma unroll
    for (int p = 0; p < S::v_pieces; ++p)
#pragma unroll
      for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int i = 0; i < S::v_cols; i += 2)
          *reinterpret_cast<float2*>(s_o + (warp * kRowsM + g + 8 * r) * kPitch + column(p, f) + i) =
              by == 0.f ? make_float2(0.f, 0.f) : make_float2(o[p * S::v_cols + i][2 * r + f] * by, o[p * S::v_cols + i + 1][2 * r + f] * by);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < min(kRowsM, rows - row0) * (kD / 2); e += 32 * kWarps) {
    const int r = e / (kD / 2), d = e % (kD / 2) * 2, row = row0 + r;
    if (d >= a.D) continue;
    float all = kNone, sum = 0.f, x = 0.f, y = 0.f;
    for (int w = 0; w < kWarps; ++w) all = fmaxf(all, s_m[w][r]);
    for (int w = 0; w < kWarps; ++w) {
      sum += s_m[w][r] == kNone ? 0.f : s_l[w][r] * ex2(s_m[w][r] - all);
      x += s_o[(w * kRowsM + r) * kPitch + d];
      y += s_o[(w * kRowsM + r) * kPitch + d + 1];
    }
    if (!whole) {
      const long long at_part = (unit * plan.splits + blockIdx.y) * kRowsM + r;
      *reinterpret_cast<float2*>(part + at_part * kD + d) = make_float2(x, y);
      if (d == 0) *reinterpret_cast<float2*>(part_ml + 2 * at_part) = make_float2(all, sum);
      continue;
    }
    const int i = row / R, h = kh * R + row % R;
    const float w = sum > 0.f ? 1.f / sum : 0.f;
    const uint32_t v = pack_bf16(x * w, y * w);
    *reinterpret_cast<uint32_t*>(at_out(a.o, seq, i, h) + d) = v;
    if (a.rest.p != nullptr) *reinterpret_cast<uint32_t*>(at_out(a.rest, seq, i, h) + d) = rest_of(x * w, y * w, v);
    if (a.lse != nullptr && d == 0) a.lse[h * q_rows + (long long)seq * a.rq.T + i] = sum > 0.f ? all + log2f(sum) : CUDART_INF_F;
  }
}

// Adds a row's splits where the first had not all of it: a block per row, a thread per four columns and turn, up to 16 of them, which
// take splits in turn.  What it costs is waiting for memory, so that a thread has eight loads on the way before it knows their weights;
// the turns' sums are added in order.  74 splits of 8 rows x 8 pairs of a sequence and a key head, cold: 5.6 us (two columns per thread,
// one load after another, 20 us).
constexpr int kMaxTurns = 16, kAhead = 8, kMaxSplits = 1024;
template <int kD>
__global__ void __launch_bounds__(kMaxTurns * kD / 4) attention_few_join_kernel(const __grid_constant__ AttnArgs a, const FewPlan plan,
                                                                             const float* __restrict__ part, const float* __restrict__ part_ml) {
  pdl_sync();
  constexpr int kQuads = kD / 4;
  const int threads = blockDim.x, turns = threads / kQuads;
  __shared__ float4 s_sum[kMaxTurns][kQuads];
  __shared__ float2 s_ml[kMaxSplits];                  // of a split: its largest score, then its weight; its sum of weights
  __shared__ float s_max[kMaxTurns * kQuads / 32], s_l[kMaxTurns];
  const int R = a.H / a.G, rows = a.rq.T * R;
  const unsigned unit = blockIdx.x, rest_of_unit = unit / plan.row_blocks;
  const int r = blockIdx.y, row0 = (int)(unit - rest_of_unit * plan.row_blocks) * kRowsM, row = row0 + r;
  if (row >= rows) return;
  const int seq = (int)(rest_of_unit / a.G), kh = (int)(rest_of_unit - (unsigned)seq * a.G);
  const Span qs = span_of(a.rq, seq), ks = span_of(a.rk, seq);
  const int last = min((min(rows, row0 + kRowsM) - 1) / R, qs.n - 1);
  const int vis = row0 / R <= last ? keys_seen(a, seq, last, qs.n, ks.n) : 0;
  if (vis <= plan.chunk) return;
  const int n = (vis + plan.chunk - 1) / plan.chunk;
  const int quad = threadIdx.x % kQuads, turn = threadIdx.x / kQuads;
  const long long first = (long long)unit * plan.splits * kRowsM + r;
  const bool there = quad * 4 < a.D;
  float4 v[kAhead];
  auto fetch = [&](int s0) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int s = s0 + k * turns;
      v[k] = there && s < n ? *reinterpret_cast<const float4*>(part + (first + (long long)s * kRowsM) * kD + quad * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  };
  fetch(turn);
  float all = kNone, sum = 0.f;
  for (int s = threadIdx.x; s < n; s += threads) {
    s_ml[s] = *reinterpret_cast<const float2*>(part_ml + 2 * (first + (long long)s * kRowsM));
    all = fmaxf(all, s_ml[s].x);
  }
  for (int o = 16; o > 0; o >>= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, o));
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = all;
  __syncthreads();
  for (int w = 0; w < threads / 32; ++w) all = fmaxf(all, s_max[w]);
  for (int s = threadIdx.x; s < n; s += threads) s_ml[s].x = s_ml[s].x == kNone ? 0.f : ex2(s_ml[s].x - all);
  __syncthreads();
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = turn; s0 < n; s0 += kAhead * turns) {
    if (s0 != turn) fetch(s0);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int s = s0 + k * turns;
      if (s >= n) break;
      const float2 by = s_ml[s];
      sum = fmaf(by.y, by.x, sum);
      x = make_float4(fmaf(v[k].x, by.x, x.x), fmaf(v[k].y, by.x, x.y), fmaf(v[k].z, by.x, x.z), fmaf(v[k].w, by.x, x.w));
    }
  }
  s_sum[turn][quad] = x;
  if (quad == 0) s_l[turn] = sum;
  __syncthreads();
  if (turn != 0 || !there) return;
  sum = 0.f;
  x = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k = 0; k < turns; ++k) {
    const float4 y = s_sum[k][quad];
    x = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
    sum += s_l[k];
  }
  const int i = row / R, h = kh * R + row % R;
  const float w = sum > 0.f ? 1.f / sum : 0.f;
  const uint2 o = make_uint2(pack_bf16(x.x * w, x.y * w), pack_bf16(x.z * w, x.w * w));
  *reinterpret_cast<uint2*>(at_out(a.o, seq, i, h) + quad * 4) = o;
  if (a.rest.p != nullptr)
    *reinterpret_cast<uint2*>(at_out(a.rest, seq, i, h) + quad * 4) =
        make_uint2(rest_of(x.x * w, x.y * w, o.x), rest_of(x.z * w, x.w * w, o.y));
  if (a.lse != nullptr && quad == 0)
    a.lse[h * ((long long)a.B * a.rq.T) + (long long)seq * a.rq.T + i] = sum > 0.f ? all + log2f(sum) : CUDART_INF_F;
}

int few_columns(const AttnArgs& a) { return a.D <= 16 ? 16 : a.D <= 32 ? 32 : a.D <= 64 ? 64 : 128; }

FewPlan plan_of(const AttnArgs& a) {
  FewPlan p{};
  p.row_blocks = (int)(((long long)a.rq.T * (a.H / a.G) + kRowsM - 1) / kRowsM);
  const long long units = (long long)a.B * a.G * p.row_blocks;
  const int keys = a.rk.T;
  // A warp each where that fills the GPU: 512 histories of 20 to 2000 x 8 heads 126 -> 94 us, 2048 of 10 to 600 x 4 heads 119 -> 64.
  p.per_unit = keys <= 2048 && units >= 148 * 8 ? 1 : kWarps;
  p.splits = 1;
  p.chunk = keys;
  if (p.per_unit == 1) {
    // and 512 keys of long ones: a warp with 2000 that starts last ends alone.  512 histories of 20 to 2000 x 8 heads x 64 columns 94 -> 87
    // us, 300 x 4 heads 53 -> 34, 300 x 4 x 128 columns 92 -> 63; 1000 of 500 to 1100 x 4 x 64 131 -> 134, 2000 of 10 to 600 would lose 61 -> 71.
    if (keys > 1024) {
      p.chunk = 512;
      p.splits = (keys + p.chunk - 1) / p.chunk;
    }
  } else {
    const long long want = (148 * 2 + units - 1) / units;           // blocks that fill the GPU
    const long long most = (keys + 255) / 256;
    long long s = want < most ? want : most;
    // Lengths may be anything: long ones are shared, 1024 keys to a block, or a 64th (4 of 131072: 95 us, with 128 splits 101).
    const long long shares = keys > 64 * 1024 ? 64 : (keys + 1023) / 1024;
    if (s < shares && a.rk.len != nullptr) s = shares;
    if (s > kMaxSplits) s = kMaxSplits;
    p.chunk = (int)((keys + s - 1) / s + 63) / 64 * 64;
    p.splits = (keys + p.chunk - 1) / p.chunk;
  }
  return p;
}

template <int kD>
cudaError_t launch(const FewMaps& maps, const AttnArgs& a, const FewPlan& p, float* work, cudaStream_t st) {
  using S = FewShape<kD>;
  static_assert(kWarps * kRowsM * (kD + 4) * 4 <= S::smem, "the warps' results take the place of the rings");
  auto* k = a.cap > kCoarseCap ? attention_few_kernel<kD, true> : attention_few_kernel<kD, false>;
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, S::smem);      // of the current device
  if (e != cudaSuccess) return e;
  const long long units = (long long)a.B * a.G * p.row_blocks;
  float* ml = work == nullptr ? nullptr : work + units * p.splits * kRowsM * kD;
  const long long blocks = p.per_unit == 1 ? (units + kWarps - 1) / kWarps : units;
  if (units >= (1LL << 31)) return cudaErrorInvalidConfiguration;
  e = launch_pdl(k, dim3((unsigned)blocks, p.splits), dim3(32 * kWarps), S::smem, st, maps, a, p, work, ml);
  if (e != cudaSuccess || p.splits == 1) return e;
  const int rows = a.rq.T * (a.H / a.G);
  int turns = kD < 128 ? 128 / kD : 1;      // a warp at least
  while (turns < kMaxTurns && turns * kAhead < p.splits) turns *= 2;
  return launch_pdl(attention_few_join_kernel<kD>, dim3((unsigned)units, rows < kRowsM ? rows : kRowsM), dim3(turns * kD / 4), 0, st, a, p, (const float*)work,
                    (const float*)ml);
}

}  // namespace

// Where the kernels for short sequences take the call too, they start fewer warps that do more.  600000 keys in sequences of 50, 100 and
// 200, 4 heads, us of those and of these:
//   1 query    16 columns 78, 68, 65 and 109, 86, 70;  32: 113, 92, 88 and 119, 100, 83;  64: 178, 160 and 135, 111
//   50         16 columns 273, 336, 373 and 461, 324, 250;  32: 432, 440, 547 and 514, 379, 299;  64: 746, 686 and 576, 399
// and one sequence of 200 with one query, 18 and 10.
bool attention_few_takes(const AttnArgs& a) {
  const long long rows = (long long)a.rq.T * (a.H / a.G), keys = mean_length(a.rk, a.B);
  if (a.rq.off != nullptr || rows > 4 * kRowsM) return false;
  if (!attention_short_takes(a, false)) return true;
  if (tile_count(a.rq, a.B, 16) * a.H < 148 * 8) return keys > 32;
  return a.D > 32 ? keys > 24 : rows > kRowsM ? keys > 80 : a.D > 16 && keys > 160;
}

long long attention_few_floats(const AttnArgs& a) {
  const FewPlan p = plan_of(a);
  return p.splits == 1 ? 0 : (long long)a.B * a.G * p.row_blocks * p.splits * kRowsM * (few_columns(a) + 2);
}

const char* launch_attention_few(const AttnArgs& a, float* work, cudaStream_t st) {
  const FewPlan p = plan_of(a);
  const int D = few_columns(a), keys = D == 128 ? FewShape<128>::keys : FewShape<64>::keys;
  FewMaps maps;
  if (!operand_map(a.k, a.D, a.rk, a.B, a.G, keys, &maps.k) || !operand_map(a.v, a.D, a.rk, a.B, a.G, keys, &maps.v))
    return "attention: cuTensorMapEncodeTiled failed";
  cudaError_t e = D == 16   ? launch<16>(maps, a, p, work, st)
                  : D == 32 ? launch<32>(maps, a, p, work, st)
                  : D == 64 ? launch<64>(maps, a, p, work, st)
                            : launch<128>(maps, a, p, work, st);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

}  // namespace tn
