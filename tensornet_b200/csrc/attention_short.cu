// Attention within short sequences, forward and backward: a warp per 16 queries or keys of a head, up to 64 columns.
//
// A tile of 128 rows is mostly empty where sequences have 40, and a block that fills tiles, barriers and tensor memory for each is
// bound by the time that takes.  Here a warp needs none of them: its rows are the left operand of mma.sync, the others' rows come
// straight from memory (from L1 and L2 after the first reader) as right operands, and what bounds it is the number of
// instructions (0.6 of the issue slots forward, 0.5 backward) and the latency of those loads.  4096 causal sequences of 1 to 200, 4
// heads x 16 columns, with a bias: 104 us forward, 250 us backward.  The mathematics is that of the kernels for long sequences (attention_fwd.cu, attention_bwd.cu): every result has one
// owner, so sums have a fixed order.
#include <cuda_bf16.h>
#include "attention_mma.cuh"

namespace tn {

namespace {

using namespace attn;

constexpr int kWarps = 4, kM = 16;

// Right operands of 16 rows at a time, straight from memory.  The lane keeps its place in the rows and moves on by 16 of them.
template <int kD>
struct ScoreRows {      // rows as columns of the product
  using P = Pieces<kD>;
  const __nv_bfloat16* p;
  int left;             // rows behind the lane's first one, itself included
  bool there[P::k_pieces];
  __device__ __forceinline__ ScoreRows(const AttnOperand& o, int b, int first, int h, int from, int n, int D, int g, int t)
      : p(at(o, b, first + from + g, h) + t * 2 * P::k_words), left(n - from - g) {
#pragma unroll
    for (int i = 0; i < P::k_pieces; ++i) there[i] = (i * 4 + t) * 2 * P::k_words < D;
  }
  __device__ __forceinline__ void load(long long st, uint32_t (*w)[P::k_all]) const {
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int i = 0; i < P::k_pieces; ++i) {
#pragma unroll
        for (int k = 0; k < P::k_words; ++k) w[c][i * P::k_words + k] = 0u;
        if (8 * c < left && there[i]) load_words<P::k_words>(p + 8 * c * st + i * 8 * P::k_words, &w[c][i * P::k_words]);
      }
  }
  __device__ __forceinline__ void next(long long st) { p += 16 * st; left -= 16; }
};
template <int kD>
struct ValueRows {      // rows as the contraction
  using P = Pieces<kD>;
  const __nv_bfloat16* p;
  int left;
  bool there[P::v_pieces];
  __device__ __forceinline__ ValueRows(const AttnOperand& o, int b, int first, int h, int from, int n, int D, int g, int t)
      : p(at(o, b, first + from + 2 * t, h) + g * P::v_cols), left(n - from - 2 * t) {
#pragma unroll
    for (int i = 0; i < P::v_pieces; ++i) there[i] = (i * 8 + g) * P::v_cols < D;
  }
  __device__ __forceinline__ void load(long long st, uint32_t (*w)[4][P::v_words]) const {
#pragma unroll
    for (int i = 0; i < P::v_pieces; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = (e & 1) + 8 * (e >> 1);
#pragma unroll
        for (int k = 0; k < P::v_words; ++k) w[i][e][k] = 0u;
        if (row < left && there[i]) load_words<P::v_words>(p + row * st + i * 8 * P::v_cols, w[i][e]);
      }
  }
  __device__ __forceinline__ void next(long long st) { p += 16 * st; left -= 16; }
};
// Left operand: the words of rows g and g + 8
template <int kD>
__device__ __forceinline__ void row_words(const __nv_bfloat16* base, long long st, int first, int n, int D, int g, int t, uint32_t (*w)[2]) {
  using P = Pieces<kD>;
#pragma unroll
  for (int e = 0; e < 2; ++e)
#pragma unroll
    for (int p = 0; p < P::k_pieces; ++p) {
      const int x = first + g + 8 * e, d = (p * 4 + t) * 2 * P::k_words;
      uint32_t v[P::k_words] = {};
      if (x < n && d < D) load_words<P::k_words>(base + x * st + d, v);
#pragma unroll
      for (int i = 0; i < P::k_words; ++i) w[p * P::k_words + i][e] = v[i];
    }
}
template <int kD>
__device__ __forceinline__ void mma_scores(float (*s)[4], const uint32_t (*x)[2], const uint32_t (*y)[Pieces<kD>::k_all]) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    s[c][0] = s[c][1] = s[c][2] = s[c][3] = 0.f;
#pragma unroll
    for (int i = 0; i < Pieces<kD>::k_all; i += 2) {
      const uint32_t a[4] = {x[i][0], x[i][1], x[i + 1][0], x[i + 1][1]};
      mma16(s[c], a, y[c][i], y[c][i + 1]);
    }
  }
}
// The lane has of row g + 8 r the columns (8 p + 2 t + f) vc + i: acc[p vc + i][2 r + f], two runs of vc columns side by side.
// kRest: not the rounded values, but what rounding took off them
template <int kD, bool kRest = false>
__device__ __forceinline__ void store_rows(const AttnOperand& to, int b, long long first, int there, int filled, int h, int D, int g, int t,
                                           const float (*acc)[4], const float* w) {
  using P = Pieces<kD>;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int x = g + 8 * r;
    if (x >= there) continue;
    __nv_bfloat16* row = at_out(to, b, first + x, h);
#pragma unroll
    for (int p = 0; p < P::v_pieces; ++p) {
      uint32_t v[2 * P::v_words];
#pragma unroll
      for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int k = 0; k < P::v_words; ++k)
          {
            const float x0 = acc[p * P::v_cols + 2 * k][2 * r + f] * w[r], x1 = acc[p * P::v_cols + 2 * k + 1][2 * r + f] * w[r];
            const uint32_t both = pack_bf16(x0, x1);
            v[f * P::v_words + k] = x >= filled ? 0u : kRest ? rest_of(x0, x1, both) : both;
          }
      const int d = (p * 8 + 2 * t) * P::v_cols;
      if constexpr (P::v_words <= 2) {
        if (d + 2 * P::v_cols <= D) store_words<2 * P::v_words>(row + d, v);
        else if (d < D) store_words<P::v_words>(row + d, v);
      } else {
        if (d < D) store_words<4>(row + d, v);
        if (d + P::v_cols < D) store_words<4>(row + d + P::v_cols, v + 4);
      }
    }
  }
}

// A warp takes `heads` heads of its tile, one after another.
template <int kD, Cap kCap, bool kBias>
__global__ void __launch_bounds__(32 * kWarps, kD == 16 ? 6 : kD == 32 ? 4 : 3) attention_short_fwd_kernel(const __grid_constant__ AttnArgs a, unsigned tiles, unsigned heads) {
  using P = Pieces<kD>;
  pdl_sync();
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const unsigned unit = blockIdx.x * kWarps + (threadIdx.x >> 5), groups = ((unsigned)a.H + heads - 1) / heads;
  const unsigned tile_at = unit / groups;
  if (tile_at >= tiles) return;
  const int h0 = (unit - tile_at * groups) * heads, h1 = min(a.H, h0 + (int)heads), R = a.H / a.G;
  const Tile tile = tile_of<false>(a.rq, a.B, kM, (int)tile_at);
  if (!tile.any) return;
  Span qs{tile.rows.b, tile.rows.first, 0}, ks{0, 0, 0};
  if (tile.seq >= 0) {
    qs = span_of(a.rq, tile.seq);
    ks = span_of(a.rk, tile.seq);
  }
  const int x0 = tile.first;
  // keys_seen grows with the query
  const int vis = x0 < qs.n ? keys_seen(a, tile.seq, min(x0 + kM, qs.n) - 1, qs.n, ks.n) : 0;
  const int least = x0 + kM <= qs.n ? keys_seen(a, tile.seq, x0, qs.n, ks.n) : 0;
  int lim[2];            // from the lane's first column on
  float row[2];          // the place of its rows, less its first column
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int x = x0 + g + 8 * e;
    lim[e] = (x < qs.n ? keys_seen(a, tile.seq, x, qs.n, ks.n) : 0) - 2 * t;
    row[e] = (float)(place_of(a, x, qs.n, ks.n) - 2 * t);
  }
  const float cs = kCap ? a.scale / a.cap : a.scale * kLog2e, cap2 = a.cap * kLog2e;
  const long long q_rows = flat_rows(a.rq, a.B), flat = (a.rq.off ? 0 : (long long)qs.b * a.rq.T) + qs.first + x0 + g;
  for (int h = h0; h < h1; ++h) {
    const float slope2 = kBias ? -a.slopes[h] * kLog2e : 0.f;
    uint32_t q[P::k_all][2];
    row_words<kD>(at(a.q, qs.b, qs.first, h), a.q.st, x0, qs.n, a.D, g, t, q);
    ScoreRows<kD> k(a.k, ks.b, ks.first, h / R, 0, vis, a.D, g, t);
    ValueRows<kD> v(a.v, ks.b, ks.first, h / R, 0, vis, a.D, g, t);
    float o[P::products][4];
#pragma unroll
    for (int i = 0; i < P::products; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[2] = {kNone, kNone};
    float2 l[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
    uint32_t kw[2][P::k_all];
    k.load(a.k.st, kw);
    for (int j0 = 0; j0 < vis; j0 += 16) {
      uint32_t vw[P::v_pieces][4][P::v_words];
      v.load(a.v.st, vw);
      v.next(a.v.st);
      float2 s[2][2];      // product (8 columns), row
      mma_scores<kD>(reinterpret_cast<float(*)[4]>(s), q, kw);
      k.next(a.k.st);
      k.load(a.k.st, kw);      // (nothing behind the last)
      float top[2] = {kNone, kNone};
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float2 x = s[c][r];
          if (kCap) {
            x = mul2(x, both(cs));
            x = mul2(tanh_any<kCap>(x), both(cap2));
          }
          if (kBias) {
            const float away = row[r] - (float)(j0 + 8 * c);
            const float2 bias = make_float2(slope2 * fabsf(away), slope2 * fabsf(away - 1.f));
            x = kCap ? add2(x, bias) : fma2(x, both(cs), bias);
          }
          if (!kCap && !kBias) x = mul2(x, both(cs));
          if (j0 + 16 > least) {
            const int there = lim[r] - j0 - 8 * c;
            x.x = there > 0 ? x.x : kNone;
            x.y = there > 1 ? x.y : kNone;
          }
          s[c][r] = x;
          top[r] = max3(top[r], x.x, x.y);
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
          l[r] = mul2(l[r], both(by));
#pragma unroll
          for (int i = 0; i < P::products; ++i) { o[i][2 * r] *= by; o[i][2 * r + 1] *= by; }
        }
      }
      uint32_t p[4];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float2 ref = both(m[r] == kNone ? 0.f : -m[r]);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float2 x = add2(s[c][r], ref);
          x = make_float2(ex2(x.x), ex2(x.y));
          l[r] = add2(l[r], x);
          p[2 * c + r] = pack_bf16(x.x, x.y);
        }
      }
#pragma unroll
      for (int pc = 0; pc < P::v_pieces; ++pc) mma_values<P::v_words>(o + pc * P::v_cols, p, vw[pc]);
    }
    float w[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float sum = l[r].x + l[r].y;
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      w[r] = sum > 0.f ? __fdividef(1.f, sum) : 0.f;
      if (a.lse != nullptr && t == 0 && x0 + g + 8 * r < qs.n) a.lse[h * q_rows + flat + 8 * r] = sum > 0.f ? m[r] + __log2f(sum) : CUDART_INF_F;
    }
    store_rows<kD>(a.o, tile.rows.b, tile.rows.first + x0, tile.rows.n - x0, qs.n - x0, h, a.D, g, t, o, w);
    if (a.rest.p != nullptr) store_rows<kD, true>(a.rest, tile.rows.b, tile.rows.first + x0, tile.rows.n - x0, qs.n - x0, h, a.D, g, t, o, w);
  }
}

// kKeys: the warp owns keys; see attention_bwd.cu for X and Y
template <int kD, Cap kCap, bool kBias, bool kKeys>
__device__ __forceinline__ void short_bwd(const AttnArgs& a, int tile_at, int head0, int head1) {
  using P = Pieces<kD>;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const Tile tile = tile_of<false>(kKeys ? a.rk : a.rq, a.B, kM, tile_at);
  if (!tile.any) return;
  Span qs{tile.rows.b, tile.rows.first, 0}, ks = qs;
  if (tile.seq >= 0) {
    qs = span_of(a.rq, tile.seq);
    ks = span_of(a.rk, tile.seq);
  }
  const Span& xs = kKeys ? ks : qs;
  const Span& ys = kKeys ? qs : ks;
  const int x0 = tile.first, R = a.H / a.G, shift = ks.n - qs.n;
  int lo = 0, hi = 0, all_lo = 0, all_hi = 0;      // rows of Y that rows of X meet, and where all meet all
  if (x0 < xs.n) {
    const int last = min(x0 + kM, xs.n) - 1;
    if (kKeys) {
      lo = first_query(a, tile.seq, x0, qs.n, ks.n) & ~15;
      hi = all_hi = qs.n;
      all_lo = first_query(a, tile.seq, last, qs.n, ks.n);
    } else {
      hi = keys_seen(a, tile.seq, last, qs.n, ks.n);
      all_hi = x0 + kM <= qs.n ? keys_seen(a, tile.seq, x0, qs.n, ks.n) : 0;
    }
  }
  const long long q_rows = flat_rows(a.rq, a.B), q_flat = (a.rq.off ? 0 : (long long)qs.b * a.rq.T) + qs.first;
  // from the lane's first column on; keys: the queries [meet, hi) see them; queries: keys [0, meet) are seen
  int meet[2];
  float row[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int x = x0 + g + 8 * e;
    meet[e] = (x >= xs.n ? 0 : kKeys ? first_query(a, tile.seq, x, qs.n, ks.n) : keys_seen(a, tile.seq, x, qs.n, ks.n)) - 2 * t;
    row[e] = (float)(!kKeys ? place_of(a, x, qs.n, ks.n) - 2 * t : a.newest ? x - (ks.n - 1) : x - shift - 2 * t);
  }
  const float cs = kCap ? a.scale / a.cap : a.scale * kLog2e, cap2 = a.cap * kLog2e;
  const AttnOperand &o1 = kKeys ? a.q : a.k, &o2 = kKeys ? a.go : a.v;
  for (int head = head0; head < head1; ++head) {
    uint32_t x1[P::k_all][2], x2[P::k_all][2];
    const AttnOperand &r1 = kKeys ? a.k : a.q, &r2 = kKeys ? a.v : a.go;
    row_words<kD>(at(r1, xs.b, xs.first, head), r1.st, x0, xs.n, a.D, g, t, x1);
    row_words<kD>(at(r2, xs.b, xs.first, head), r2.st, x0, xs.n, a.D, g, t, x2);
    float lse[2] = {0.f, 0.f}, delta[2] = {0.f, 0.f};      // negative
    if (!kKeys)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (x0 + g + 8 * e < qs.n) {
          const long long i = head * q_rows + q_flat + x0 + g + 8 * e;
          lse[e] = -a.lse[i];
          delta[e] = -a.delta[i];
        }
    float acc1[P::products][4], acc2[kKeys ? P::products : 1][4];
#pragma unroll
    for (int i = 0; i < P::products; ++i) acc1[i][0] = acc1[i][1] = acc1[i][2] = acc1[i][3] = 0.f;
    if (kKeys)
#pragma unroll
      for (int i = 0; i < P::products; ++i) acc2[i][0] = acc2[i][1] = acc2[i][2] = acc2[i][3] = 0.f;
    for (int hh = 0; hh < (kKeys ? R : 1); ++hh) {
      const int h = kKeys ? head * R + hh : head, hy = kKeys ? h : head / R;
      const float slope2 = kBias ? -a.slopes[h] * kLog2e : 0.f;
      ScoreRows<kD> s1(o1, ys.b, ys.first, hy, lo, hi, a.D, g, t), s2(o2, ys.b, ys.first, hy, lo, hi, a.D, g, t);
      ValueRows<kD> v1(o1, ys.b, ys.first, hy, lo, hi, a.D, g, t), v2(o2, ys.b, ys.first, hy, lo, hi, a.D, g, t);
      const float *lse_y = a.lse + h * q_rows + q_flat + 2 * t, *delta_y = a.delta + h * q_rows + q_flat + 2 * t;
      for (int y0 = lo; y0 < hi; y0 += 16) {
        uint32_t w1[2][P::k_all], w2[2][P::k_all], u1[P::v_pieces][4][P::v_words], u2[kKeys ? P::v_pieces : 1][4][P::v_words];
        s1.load(o1.st, w1);
        s2.load(o2.st, w2);
        s1.next(o1.st);
        s2.next(o2.st);
        float2 ly[2], dy[2];
        if (kKeys)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int y = y0 + 8 * c, left = hi - y - 2 * t;
            ly[c] = make_float2(left > 0 ? -lse_y[y] : 0.f, left > 1 ? -lse_y[y + 1] : 0.f);
            dy[c] = make_float2(left > 0 ? -delta_y[y] : 0.f, left > 1 ? -delta_y[y + 1] : 0.f);
          }
        v1.load(o1.st, u1);
        v1.next(o1.st);
        if (kKeys) {
          v2.load(o2.st, u2);
          v2.next(o2.st);
        }
        float2 s[2][2], d[2][2];
        mma_scores<kD>(reinterpret_cast<float(*)[4]>(s), x1, w1);
        mma_scores<kD>(reinterpret_cast<float(*)[4]>(d), x2, w2);
        const bool masked = y0 < all_lo || y0 + 16 > all_hi;
        uint32_t da[4], dr[4], pa[4];      // ds and what rounding took off it: products cost little here, and few terms average little out
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float2 lg = kKeys ? ly[c] : both(lse[r]), dl = kKeys ? dy[c] : both(delta[r]);
            float2 arg, slope;
            if (kCap) {
              const float2 y = mul2(s[c][r], both(cs));
              const float2 th = tanh_any<kCap>(y);
              arg = fma2(th, both(cap2), lg);
              slope = fma2(mul2(th, both(-1.f)), th, both(1.f));
            } else {
              arg = fma2(s[c][r], both(cs), lg);
            }
            if (kBias) {
              const float at_y = (float)(y0 + 8 * c), away = kKeys ? fmaf(-a.step, at_y, row[r]) : row[r] - at_y;
              arg = add2(arg, make_float2(slope2 * fabsf(away), slope2 * fabsf(away - (kKeys ? a.step : 1.f))));
            }
            float2 p = make_float2(ex2(arg.x), ex2(arg.y));
            float2 ds = mul2(p, add2(d[c][r], dl));
            if (kCap) ds = mul2(ds, slope);
            if (masked) {
              const int y = y0 + 8 * c, n = (kKeys ? hi - 2 * t : meet[r]) - y, k = kKeys ? meet[r] - y : 0;      // of the lane's columns, [k, n)
              if (!(n > 0 && k <= 0)) p.x = ds.x = 0.f;
              if (!(n > 1 && k <= 1)) p.y = ds.y = 0.f;
            }
            da[2 * c + r] = pack_bf16(ds.x, ds.y);
            dr[2 * c + r] = rest_of(ds.x, ds.y, da[2 * c + r]);
            if (kKeys) pa[2 * c + r] = pack_bf16(p.x, p.y);
          }
#pragma unroll
        for (int pc = 0; pc < P::v_pieces; ++pc) {
          mma_values<P::v_words>(acc1 + pc * P::v_cols, da, u1[pc]);
          mma_values<P::v_words>(acc1 + pc * P::v_cols, dr, u1[pc]);
        }
        if (kKeys)
#pragma unroll
          for (int pc = 0; pc < P::v_pieces; ++pc) mma_values<P::v_words>(acc2 + pc * P::v_cols, pa, u2[pc]);
      }
    }
    const float scales[2] = {a.scale, a.scale}, ones[2] = {1.f, 1.f};
    const long long first = tile.rows.first + x0;
    const int there = tile.rows.n - x0, filled = xs.n - x0;
    store_rows<kD>(kKeys ? a.gk : a.gq, tile.rows.b, first, there, filled, head, a.D, g, t, acc1, scales);
    if (kKeys) store_rows<kD>(a.gv, tile.rows.b, first, there, filled, head, a.D, g, t, acc2, ones);
  }
}

// The first key_units warps own keys, the others queries.
template <int kD, Cap kCap, bool kBias>
__global__ void __launch_bounds__(32 * kWarps, kD == 16 ? 4 : kD == 32 ? 3 : 2)
attention_short_bwd_kernel(const __grid_constant__ AttnArgs a, unsigned key_units, unsigned units, unsigned key_heads, unsigned heads) {
  pdl_sync();
  const unsigned unit = blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (unit >= units) return;
  if (unit < key_units) {
    const unsigned groups = ((unsigned)a.G + key_heads - 1) / key_heads, tile = unit / groups, h0 = (unit - tile * groups) * key_heads;
    short_bwd<kD, kCap, kBias, true>(a, (int)tile, (int)h0, min(a.G, (int)(h0 + key_heads)));
  } else {
    const unsigned at = unit - key_units, groups = ((unsigned)a.H + heads - 1) / heads, tile = at / groups, h0 = (at - tile * groups) * heads;
    short_bwd<kD, kCap, kBias, false>(a, (int)tile, (int)h0, min(a.H, (int)(h0 + heads)));
  }
}

// Heads that a warp takes of its tile: finding the tile costs as much as a step or two, but every SM wants some 32 warps, and again as
// many in turn.
unsigned heads_of(long long tiles, int H) {
  unsigned n = 1;
  while (n < 8 && n < (unsigned)H && tiles * ((H + 2 * n - 1) / (2 * n)) >= 148 * 64) n *= 2;
  return n;
}

template <int kD, Cap kCap, bool kBias>
cudaError_t launch_fwd(const AttnArgs& a, cudaStream_t st) {
  const long long tiles = tile_count(a.rq, a.B, kM);
  const unsigned heads = heads_of(tiles, a.H);
  const long long units = tiles * ((a.H + heads - 1) / heads);
  if (units >= (1LL << 31)) return cudaErrorInvalidConfiguration;
  return launch_pdl(attention_short_fwd_kernel<kD, kCap, kBias>, dim3((unsigned)((units + kWarps - 1) / kWarps)), dim3(32 * kWarps), 0, st, a,
                    (unsigned)tiles, heads);
}
template <int kD, Cap kCap, bool kBias>
cudaError_t launch_bwd(const AttnArgs& a, cudaStream_t st) {
  const long long key_tiles = tile_count(a.rk, a.B, kM), tiles = tile_count(a.rq, a.B, kM);
  const unsigned key_heads = heads_of(key_tiles, a.G), heads = heads_of(tiles, a.H);
  const long long key_units = key_tiles * ((a.G + key_heads - 1) / key_heads), units = key_units + tiles * ((a.H + heads - 1) / heads);
  if (units >= (1LL << 31)) return cudaErrorInvalidConfiguration;
  return launch_pdl(attention_short_bwd_kernel<kD, kCap, kBias>, dim3((unsigned)((units + kWarps - 1) / kWarps)), dim3(32 * kWarps), 0, st, a,
                    (unsigned)key_units, (unsigned)units, key_heads, heads);
}
template <int kD>
cudaError_t launch(bool fwd, const AttnArgs& a, cudaStream_t st) {
  return with_cap(a, [&](auto cap) {
    constexpr Cap kCap = decltype(cap)::value;
    if (a.slopes) return fwd ? launch_fwd<kD, kCap, true>(a, st) : launch_bwd<kD, kCap, true>(a, st);
    return fwd ? launch_fwd<kD, kCap, false>(a, st) : launch_bwd<kD, kCap, false>(a, st);
  });
}
const char* told(cudaError_t e) {
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

}  // namespace

// By the mean length, which is what the host knows of packed sequences.  200000 tokens, 4 heads, causal, us of these kernels and of those
// for long sequences:
//   forward   16 columns: 200 tokens 135 and 246, 400: 205 and 293;  32: 200: 183 and 256, 400: 268 and 305;  64: 128: 233 and 252, 200: 295
//             and 265
//   backward  16 columns: 256 tokens 417 and 501, 400: 577 and 638;  32: 200: 562 and 663, 256: 632 and 545;  64: 64: 636 and 826, 100: 771
//             and 769
bool attention_short_takes(const AttnArgs& a, bool backward) {
  const int most = backward ? (a.D <= 16 ? 400 : a.D <= 32 ? 224 : 96) : (a.D <= 16 ? 512 : a.D <= 32 ? 400 : 144);
  return a.D <= 64 && mean_length(a.rq, a.B) <= most && mean_length(a.rk, a.B) <= most;
}

const char* launch_attention_short_fwd(const AttnArgs& a, cudaStream_t st) {
  return told(a.D <= 16 ? launch<16>(true, a, st) : a.D <= 32 ? launch<32>(true, a, st) : launch<64>(true, a, st));
}
const char* launch_attention_short_bwd(const AttnArgs& a, cudaStream_t st) {
  return told(a.D <= 16 ? launch<16>(false, a, st) : a.D <= 32 ? launch<32>(false, a, st) : launch<64>(false, a, st));
}

}  // namespace tn
