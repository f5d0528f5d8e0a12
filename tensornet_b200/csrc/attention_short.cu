// Attention within short sequences, forward and backward: a warp per 16 queries or keys of a head, up to 64 columns.
//
// A tile of 128 rows is mostly empty where sequences have 40, and a block that fills tiles, barriers and tensor memory for each is
// bound by the time that takes.  Here a warp needs none of them: its rows are the left operand of mma.sync, the others' rows come
// straight from memory (from L1 and L2 after the first reader) as right operands, and what bounds it is the number of
// instructions.  The mathematics is that of the kernels for long sequences (attention_fwd.cu, attention_bwd.cu): every result has one
// owner, so sums have a fixed order.
#include <cuda_bf16.h>
#include "attention_mma.cuh"

namespace tn {

namespace {

using namespace attn;

constexpr int kWarps = 4, kM = 16;

// Right operands of 16 rows from `first` on, n of them there, straight from memory
template <int kD>
__device__ __forceinline__ void score_words(const __nv_bfloat16* base, long long st, int first, int n, int D, int g, int t,
                                            uint32_t (*w)[Pieces<kD>::k_all]) {
  using P = Pieces<kD>;
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int p = 0; p < P::k_pieces; ++p) {
      const int y = first + 8 * c + g, d = (p * 4 + t) * 2 * P::k_words;
#pragma unroll
      for (int i = 0; i < P::k_words; ++i) w[c][p * P::k_words + i] = 0u;
      if (y < n && d < D) load_words<P::k_words>(base + y * st + d, &w[c][p * P::k_words]);
    }
}
template <int kD>
__device__ __forceinline__ void value_words(const __nv_bfloat16* base, long long st, int first, int n, int D, int g, int t,
                                            uint32_t (*w)[4][Pieces<kD>::v_words]) {
  using P = Pieces<kD>;
#pragma unroll
  for (int p = 0; p < P::v_pieces; ++p)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int y = first + 2 * t + (e & 1) + 8 * (e >> 1), d = (p * 8 + g) * P::v_cols;
#pragma unroll
      for (int i = 0; i < P::v_words; ++i) w[p][e][i] = 0u;
      if (y < n && d < D) load_words<P::v_words>(base + y * st + d, w[p][e]);
    }
}
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
template <int kD>
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
          v[f * P::v_words + k] = x < filled ? pack_bf16(acc[p * P::v_cols + 2 * k][2 * r + f] * w[r], acc[p * P::v_cols + 2 * k + 1][2 * r + f] * w[r]) : 0u;
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

template <int kD>
__global__ void __launch_bounds__(32 * kWarps) attention_short_fwd_kernel(const __grid_constant__ AttnArgs a, int tiles) {
  using P = Pieces<kD>;
  pdl_sync();
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const long long unit = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (unit >= (long long)tiles * a.H) return;
  const int h = (int)(unit % a.H), kh = h / (a.H / a.G);
  const Tile tile = tile_of(a.rq, a.B, kM, (int)(unit / a.H));
  if (!tile.any) return;
  Span qs{tile.rows.b, tile.rows.first, 0}, ks{0, 0, 0};
  if (tile.seq >= 0) {
    qs = span_of(a.rq, tile.seq);
    ks = span_of(a.rk, tile.seq);
  }
  const int x0 = tile.first;
  int lim[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) lim[e] = x0 + g + 8 * e < qs.n ? keys_seen(a, tile.seq, x0 + g + 8 * e, qs.n, ks.n) : 0;
  const int vis = x0 < qs.n ? keys_seen(a, tile.seq, min(x0 + kM, qs.n) - 1, qs.n, ks.n) : 0;      // keys_seen grows with the query
  const int least = x0 + kM <= qs.n ? keys_seen(a, tile.seq, x0, qs.n, ks.n) : 0;
  uint32_t q[P::k_all][2];
  row_words<kD>(at(a.q, qs.b, qs.first, h), a.q.st, x0, qs.n, a.D, g, t, q);
  const __nv_bfloat16 *k = at(a.k, ks.b, ks.first, kh), *v = at(a.v, ks.b, ks.first, kh);
  const float cs = a.cap > 0.f ? 2.f * kLog2e * a.scale / a.cap : a.scale * kLog2e, cap2 = a.cap * kLog2e;
  const float slope2 = a.slopes ? a.slopes[h] * kLog2e : 0.f;
  float o[P::products][4];
#pragma unroll
  for (int i = 0; i < P::products; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m[2] = {kNone, kNone}, l[2] = {0.f, 0.f};
  uint32_t kw[2][P::k_all];
  if (vis > 0) score_words<kD>(k, a.k.st, 0, vis, a.D, g, t, kw);
  for (int j0 = 0; j0 < vis; j0 += 16) {
    uint32_t vw[P::v_pieces][4][P::v_words];
    value_words<kD>(v, a.v.st, j0, vis, a.D, g, t, vw);
    float s[2][4];
    mma_scores<kD>(s, q, kw);
    if (j0 + 16 < vis) score_words<kD>(k, a.k.st, j0 + 16, vis, a.D, g, t, kw);
    const bool masked = j0 + 16 > least;
    float top[2] = {kNone, kNone};
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = j0 + 8 * c + 2 * t + (e & 1), r = e >> 1;
        float x = s[c][e] * cs;
        if (a.cap > 0.f) x = cap2 - __fdividef(2.f * cap2, 1.f + ex2(x));
        if (a.slopes != nullptr) x -= slope2 * fabsf((float)(x0 + g + 8 * r + ks.n - qs.n - j));
        if (masked) x = j < lim[r] ? x : kNone;
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
        if (j0 > 0)
#pragma unroll
          for (int i = 0; i < P::products; ++i) { o[i][2 * r] *= by; o[i][2 * r + 1] *= by; }
      }
    }
    const float ref[2] = {m[0] == kNone ? 0.f : m[0], m[1] == kNone ? 0.f : m[1]};
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[c][e] = ex2(s[c][e] - ref[e >> 1]);
        l[e >> 1] += s[c][e];
      }
    const uint32_t p[4] = {pack_bf16(s[0][0], s[0][1]), pack_bf16(s[0][2], s[0][3]), pack_bf16(s[1][0], s[1][1]), pack_bf16(s[1][2], s[1][3])};
#pragma unroll
    for (int pc = 0; pc < P::v_pieces; ++pc) mma_values<P::v_words>(o + pc * P::v_cols, p, vw[pc]);
  }
  float w[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    w[r] = l[r] > 0.f ? 1.f / l[r] : 0.f;
    const int x = x0 + g + 8 * r;
    if (a.lse != nullptr && t == 0 && x < qs.n)
      a.lse[h * flat_rows(a.rq, a.B) + (a.rq.off ? 0 : (long long)qs.b * a.rq.T) + qs.first + x] = l[r] > 0.f ? m[r] + log2f(l[r]) : CUDART_INF_F;
  }
  store_rows<kD>(a.o, tile.rows.b, tile.rows.first + x0, tile.rows.n - x0, qs.n - x0, h, a.D, g, t, o, w);
}

// kKeys: the warp owns keys; see attention_bwd.cu for X and Y
template <int kD, bool kKeys>
__device__ __forceinline__ void short_bwd(const AttnArgs& a, int tile_at, int head) {
  using P = Pieces<kD>;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const Tile tile = tile_of(kKeys ? a.rk : a.rq, a.B, kM, tile_at);
  if (!tile.any) return;
  Span qs{tile.rows.b, tile.rows.first, 0}, ks = qs;
  if (tile.seq >= 0) {
    qs = span_of(a.rq, tile.seq);
    ks = span_of(a.rk, tile.seq);
  }
  const Span& xs = kKeys ? ks : qs;
  const int x0 = tile.first, R = a.H / a.G;
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
  // keys: the queries [meet, nq) see them; queries: keys [0, meet) are seen
  int meet[2];
  float lse[2] = {0.f, 0.f}, delta[2] = {0.f, 0.f};
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int x = x0 + g + 8 * e;
    const bool there = x < xs.n;
    if (kKeys) {
      meet[e] = there ? first_query(a, tile.seq, x, qs.n, ks.n) : 0;
    } else {
      meet[e] = there ? keys_seen(a, tile.seq, x, qs.n, ks.n) : 0;
      if (there) {
        lse[e] = a.lse[head * q_rows + q_flat + x];
        delta[e] = a.delta[head * q_rows + q_flat + x];
      }
    }
  }
  uint32_t x1[P::k_all][2], x2[P::k_all][2];
  if (kKeys) {
    row_words<kD>(at(a.k, ks.b, ks.first, head), a.k.st, x0, ks.n, a.D, g, t, x1);
    row_words<kD>(at(a.v, ks.b, ks.first, head), a.v.st, x0, ks.n, a.D, g, t, x2);
  } else {
    row_words<kD>(at(a.q, qs.b, qs.first, head), a.q.st, x0, qs.n, a.D, g, t, x1);
    row_words<kD>(at(a.go, qs.b, qs.first, head), a.go.st, x0, qs.n, a.D, g, t, x2);
  }
  float acc1[P::products][4], acc2[kKeys ? P::products : 1][4];
#pragma unroll
  for (int i = 0; i < P::products; ++i) acc1[i][0] = acc1[i][1] = acc1[i][2] = acc1[i][3] = 0.f;
  if (kKeys)
#pragma unroll
    for (int i = 0; i < P::products; ++i) acc2[i][0] = acc2[i][1] = acc2[i][2] = acc2[i][3] = 0.f;
  const float cs = a.cap > 0.f ? 2.f * kLog2e * a.scale / a.cap : a.scale * kLog2e, cap2 = a.cap * kLog2e;
  const int shift = ks.n - qs.n;
  for (int hh = 0; hh < (kKeys ? R : 1); ++hh) {
    const int h = kKeys ? head * R + hh : head;
    const float slope2 = a.slopes ? a.slopes[h] * kLog2e : 0.f;
    const __nv_bfloat16 *y1 = kKeys ? at(a.q, qs.b, qs.first, h) : at(a.k, ks.b, ks.first, head / R);
    const __nv_bfloat16 *y2 = kKeys ? at(a.go, qs.b, qs.first, h) : at(a.v, ks.b, ks.first, head / R);
    const long long st1 = kKeys ? a.q.st : a.k.st, st2 = kKeys ? a.go.st : a.v.st;
    const float *lse_y = a.lse + h * q_rows + q_flat, *delta_y = a.delta + h * q_rows + q_flat;
    for (int y0 = lo; y0 < hi; y0 += 16) {
      uint32_t w1[2][P::k_all], w2[2][P::k_all];
      score_words<kD>(y1, st1, y0, hi, a.D, g, t, w1);
      score_words<kD>(y2, st2, y0, hi, a.D, g, t, w2);
      float ly[2][2], dy[2][2];
      if (kKeys)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int f = 0; f < 2; ++f) {
            const int y = y0 + 8 * c + 2 * t + f;
            ly[c][f] = y < hi ? lse_y[y] : 0.f;
            dy[c][f] = y < hi ? delta_y[y] : 0.f;
          }
      uint32_t u1[P::v_pieces][4][P::v_words], u2[kKeys ? P::v_pieces : 1][4][P::v_words];
      value_words<kD>(y1, st1, y0, hi, a.D, g, t, u1);
      if (kKeys) value_words<kD>(y2, st2, y0, hi, a.D, g, t, u2);
      float s[2][4], d[2][4];
      mma_scores<kD>(s, x1, w1);
      mma_scores<kD>(d, x2, w2);
      const bool masked = y0 < all_lo || y0 + 16 > all_hi;
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = e >> 1, f = e & 1, x = x0 + g + 8 * r, y = y0 + 8 * c + 2 * t + f;
          const float lg = kKeys ? ly[c][f] : lse[r], dl = kKeys ? dy[c][f] : delta[r];
          float arg, slope = 1.f;
          if (a.cap > 0.f) {
            const float tt = __fdividef(1.f, 1.f + ex2(s[c][e] * cs));
            arg = cap2 - 2.f * cap2 * tt - lg;
            slope = 4.f * tt * (1.f - tt);
          } else {
            arg = fmaf(s[c][e], cs, -lg);
          }
          if (a.slopes != nullptr) arg -= slope2 * fabsf((float)(kKeys ? y + shift - x : x + shift - y));
          float p = ex2(arg), ds = p * (d[c][e] - dl) * slope;
          if (masked && !(kKeys ? y >= meet[r] && y < hi : y < meet[r])) p = ds = 0.f;
          s[c][e] = p;
          d[c][e] = ds;
        }
      const uint32_t da[4] = {pack_bf16(d[0][0], d[0][1]), pack_bf16(d[0][2], d[0][3]), pack_bf16(d[1][0], d[1][1]), pack_bf16(d[1][2], d[1][3])};
#pragma unroll
      for (int pc = 0; pc < P::v_pieces; ++pc) mma_values<P::v_words>(acc1 + pc * P::v_cols, da, u1[pc]);
      if (kKeys) {
        const uint32_t pa[4] = {pack_bf16(s[0][0], s[0][1]), pack_bf16(s[0][2], s[0][3]), pack_bf16(s[1][0], s[1][1]), pack_bf16(s[1][2], s[1][3])};
#pragma unroll
        for (int pc = 0; pc < P::v_pieces; ++pc) mma_values<P::v_words>(acc2 + pc * P::v_cols, pa, u2[pc]);
      }
    }
  }
  const float scales[2] = {a.scale, a.scale}, ones[2] = {1.f, 1.f};
  const long long first = tile.rows.first + x0;
  const int there = tile.rows.n - x0, filled = xs.n - x0;
  store_rows<kD>(kKeys ? a.gk : a.gq, tile.rows.b, first, there, filled, head, a.D, g, t, acc1, scales);
  if (kKeys) store_rows<kD>(a.gv, tile.rows.b, first, there, filled, head, a.D, g, t, acc2, ones);
}

// The first key_units warps own keys, the others queries.
template <int kD>
__global__ void __launch_bounds__(32 * kWarps) attention_short_bwd_kernel(const __grid_constant__ AttnArgs a, long long key_units, long long units) {
  pdl_sync();
  const long long unit = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (unit >= units) return;
  if (unit < key_units) short_bwd<kD, true>(a, (int)(unit / a.G), (int)(unit % a.G));
  else short_bwd<kD, false>(a, (int)((unit - key_units) / a.H), (int)((unit - key_units) % a.H));
}

template <int kD>
cudaError_t launch_fwd(const AttnArgs& a, cudaStream_t st) {
  const long long tiles = tile_count(a.rq, a.B, kM), blocks = (tiles * a.H + kWarps - 1) / kWarps;
  if (blocks >= (1LL << 31)) return cudaErrorInvalidConfiguration;
  return launch_pdl(attention_short_fwd_kernel<kD>, dim3((unsigned)blocks), dim3(32 * kWarps), 0, st, a, (int)tiles);
}
template <int kD>
cudaError_t launch_bwd(const AttnArgs& a, cudaStream_t st) {
  const long long key_units = tile_count(a.rk, a.B, kM) * a.G, units = key_units + tile_count(a.rq, a.B, kM) * a.H;
  const long long blocks = (units + kWarps - 1) / kWarps;
  if (blocks >= (1LL << 31)) return cudaErrorInvalidConfiguration;
  return launch_pdl(attention_short_bwd_kernel<kD>, dim3((unsigned)blocks), dim3(32 * kWarps), 0, st, a, key_units, units);
}
const char* told(cudaError_t e) {
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

// the mean length where the host knows no more
long long length_of(const AttnRows& r, int B) { return r.off ? r.T / (B > 0 ? B : 1) : r.T; }

}  // namespace

bool attention_short_takes(const AttnArgs& a) { return a.D <= 64 && length_of(a.rq, a.B) <= kAttnShort && length_of(a.rk, a.B) <= kAttnShort; }

const char* launch_attention_short_fwd(const AttnArgs& a, cudaStream_t st) {
  return told(a.D <= 16 ? launch_fwd<16>(a, st) : a.D <= 32 ? launch_fwd<32>(a, st) : launch_fwd<64>(a, st));
}
const char* launch_attention_short_bwd(const AttnArgs& a, cudaStream_t st) {
  return told(a.D <= 16 ? launch_bwd<16>(a, st) : a.D <= 32 ? launch_bwd<32>(a, st) : launch_bwd<64>(a, st));
}

}  // namespace tn
