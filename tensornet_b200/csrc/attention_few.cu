// Attention of a few queries against many keys, forward: up to 16 rows, a query head's query each, that share a key head.
//
// What bounds it is reading keys and values once.  A warp takes 16 or 32 keys at a time with a softmax of its own and no shared
// memory: products are mma.sync of 16 rows (at these rates far from what bounds it), and both operands come from memory in the
// layout that the instruction wants.
//   * scores: the contraction may go over the columns in any order that both sides share.  A lane of group g = lane / 4, t = lane % 4
//     loads the 16 bytes of key g at column 8 t of 32: four words, the right operand of two products whose k are those columns.
//   * values: lane (g, t) loads the 16 bytes of keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9 at column 8 g of 64.  Words of two keys,
//     interleaved by byte permutation, are the right operand of eight products; product i has columns 8 g + i.
// Rows of 16 or 32 columns take pieces of 4 or 8 bytes in the same way.
// A sequence's keys are split over warps, blocks or both; what the blocks have of a row is brought to one reference and added by a
// second kernel, in a fixed order.
#include <cuda_bf16.h>
#include "attention_tc.cuh"

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

__device__ __forceinline__ void mma16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// kWords 32-bit words at p, or zeros
template <int kWords>
__device__ __forceinline__ void load_words(const __nv_bfloat16* p, bool there, uint32_t* w) {
  if constexpr (kWords == 4) {
    const uint4 v = there ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else if constexpr (kWords == 2) {
    const uint2 v = there ? __ldg(reinterpret_cast<const uint2*>(p)) : make_uint2(0, 0);
    w[0] = v.x; w[1] = v.y;
  } else {
    w[0] = there ? __ldg(reinterpret_cast<const uint32_t*>(p)) : 0u;
  }
}

template <int kD>
struct FewShape {
  static constexpr int keys = kD == 128 ? 16 : 32;                    // of a step
  static constexpr int k_words = kD == 16 ? 2 : 4, k_pieces = kD == 16 ? 1 : kD / 32;
  static constexpr int v_words = kD >= 64 ? 4 : kD / 16, v_pieces = kD >= 64 ? kD / 64 : 1;
  static constexpr int v_cols = 2 * v_words;                          // columns of a piece
};

// part: [unit][split][16][kD] sums and [unit][split][2][16] references and sums of weights, where there are several splits
template <int kD>
__global__ void __launch_bounds__(32 * kWarps) attention_few_kernel(const __grid_constant__ AttnArgs a, const FewPlan plan, float* __restrict__ part,
                                                                    float* __restrict__ part_ml) {
  using S = FewShape<kD>;
  constexpr int kTilesN = S::keys / 8;
  pdl_sync();
  __shared__ float s_m[kWarps][kRowsM], s_l[kWarps][kRowsM];
  __shared__ __align__(16) float s_o[kWarps][kRowsM][kD];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int R = a.H / a.G, rows = a.rq.T * R;
  const long long units = (long long)a.B * a.G * plan.row_blocks;
  const bool alone = plan.per_unit == 1;
  const long long unit = alone ? (long long)blockIdx.x * kWarps + warp : blockIdx.x;
  if (unit >= units) return;
  const int rb = (int)(unit % plan.row_blocks), kh = (int)(unit / plan.row_blocks % a.G), seq = (int)(unit / plan.row_blocks / a.G);
  const Span qs = span_of(a.rq, seq), ks = span_of(a.rk, seq);
  const int row0 = rb * kRowsM;
  // row r of the unit: query (row0 + r) / R, query head kh * R + (row0 + r) % R
  int lim[2], place[2];
  float slope2[2];
  const __nv_bfloat16* q_at[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = row0 + g + 8 * e, i = r / R, h = kh * R + r % R;
    const bool there = r < rows && i < qs.n;
    lim[e] = there ? keys_seen(a, seq, i, qs.n, ks.n) : 0;
    place[e] = i + ks.n - qs.n;
    slope2[e] = there && a.slopes ? a.slopes[h] * kLog2e : 0.f;
    q_at[e] = there ? at(a.q, qs.b, i, h) : nullptr;
  }
  int vis = max(lim[0], lim[1]);
  for (int o = 16; o > 0; o >>= 1) vis = max(vis, __shfl_xor_sync(0xffffffffu, vis, o));
  const int from = blockIdx.y * plan.chunk, to = min(vis, from + plan.chunk);

  uint32_t q[S::k_pieces * S::k_words][2];      // words of rows g and g + 8
#pragma unroll
  for (int p = 0; p < S::k_pieces; ++p)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int d = (p * 4 + t) * 2 * S::k_words;
      uint32_t w[S::k_words];
      load_words<S::k_words>(q_at[e] + d, q_at[e] != nullptr && d < a.D, w);
#pragma unroll
      for (int i = 0; i < S::k_words; ++i) q[p * S::k_words + i][e] = w[i];
    }

  uint32_t kw[kTilesN][S::k_pieces * S::k_words];
  uint32_t vw[S::keys / 16][4][S::v_pieces * S::v_words];
  const __nv_bfloat16* k_base = at(a.k, ks.b, ks.first, kh);
  const __nv_bfloat16* v_base = at(a.v, ks.b, ks.first, kh);
  auto load_k = [&](int j0) {
#pragma unroll
    for (int n = 0; n < kTilesN; ++n)
#pragma unroll
      for (int p = 0; p < S::k_pieces; ++p) {
        const int j = j0 + n * 8 + g, d = (p * 4 + t) * 2 * S::k_words;
        load_words<S::k_words>(k_base + j * a.k.st + d, j < to && d < a.D, &kw[n][p * S::k_words]);
      }
  };
  auto load_v = [&](int j0) {
#pragma unroll
    for (int n = 0; n < S::keys / 16; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int p = 0; p < S::v_pieces; ++p) {
          const int j = j0 + n * 16 + 2 * t + (e & 1) + (e >> 1) * 8, d = (p * 8 + g) * S::v_cols;
          load_words<S::v_words>(v_base + j * a.v.st + d, j < to && d < a.D, &vw[n][e][p * S::v_words]);
        }
  };

  float o[S::v_pieces * S::v_cols][4];
#pragma unroll
  for (int i = 0; i < S::v_pieces * S::v_cols; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m[2] = {kNone, kNone}, l[2] = {0.f, 0.f};
  const int stride = S::keys * plan.per_unit;
  const int j_first = from + (alone ? 0 : warp * S::keys);
  const float cs = a.cap > 0.f ? 2.f * kLog2e * a.scale / a.cap : a.scale * kLog2e;
  const float cap2 = a.cap * kLog2e;
  if (j_first < to) { load_k(j_first); load_v(j_first); }
  for (int j0 = j_first; j0 < to; j0 += stride) {
    float s[kTilesN][4];
#pragma unroll
    for (int n = 0; n < kTilesN; ++n) {
      s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
      for (int w = 0; w < S::k_pieces * S::k_words; w += 2) {
        const uint32_t aw[4] = {q[w][0], q[w][1], q[w + 1][0], q[w + 1][1]};
        mma16(s[n], aw, kw[n][w], kw[n][w + 1]);
      }
    }
    if (j0 + stride < to) load_k(j0 + stride);
    float top[2] = {kNone, kNone};
#pragma unroll
    for (int n = 0; n < kTilesN; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = j0 + n * 8 + 2 * t + (e & 1), r = e >> 1;
        float x = s[n][e] * cs;
        if (a.cap > 0.f) x = cap2 - __fdividef(2.f * cap2, 1.f + ex2(x));
        if (a.slopes != nullptr) x -= slope2[r] * fabsf((float)(place[r] - j));
        x = j < min(lim[r], to) ? x : kNone;
        s[n][e] = x;
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
#pragma unroll
    for (int n = 0; n < kTilesN; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = e >> 1;
        s[n][e] = ex2(s[n][e] - (m[r] == kNone ? 0.f : m[r]));
        l[r] += s[n][e];
      }
#pragma unroll
    for (int n = 0; n < S::keys / 16; ++n) {
      const uint32_t p[4] = {pack_bf16(s[2 * n][0], s[2 * n][1]), pack_bf16(s[2 * n][2], s[2 * n][3]), pack_bf16(s[2 * n + 1][0], s[2 * n + 1][1]),
                             pack_bf16(s[2 * n + 1][2], s[2 * n + 1][3])};
#pragma unroll
      for (int i = 0; i < S::v_pieces * S::v_words; ++i) {
        const uint32_t lo0 = __byte_perm(vw[n][0][i], vw[n][1][i], 0x5410), hi0 = __byte_perm(vw[n][0][i], vw[n][1][i], 0x7632);
        const uint32_t lo1 = __byte_perm(vw[n][2][i], vw[n][3][i], 0x5410), hi1 = __byte_perm(vw[n][2][i], vw[n][3][i], 0x7632);
        mma16(o[2 * i], p, lo0, lo1);
        mma16(o[2 * i + 1], p, hi0, hi1);
      }
    }
    if (j0 + stride < to) load_v(j0 + stride);
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
  }

  // Lane (g, t) has of row g + 8 r the columns (p 8 + 2 t + f) v_cols + i, f < 2, i < v_cols: value o[p v_cols + i][2 r + f].
  const long long q_rows = (long long)a.B * a.rq.T;
  if (alone) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = row0 + g + 8 * r;
      if (row >= rows) continue;
      const int i = row / R, h = kh * R + row % R;
      const float w = l[r] > 0.f ? 1.f / l[r] : 0.f;
      __nv_bfloat16* out = at_out(a.o, seq, i, h);
#pragma unroll
      for (int p = 0; p < S::v_pieces; ++p)
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          const int d = (p * 8 + 2 * t + f) * S::v_cols;
          if (d >= a.D) continue;
          uint32_t v[S::v_words];
#pragma unroll
          for (int k = 0; k < S::v_words; ++k)
            v[k] = pack_bf16(o[p * S::v_cols + 2 * k][2 * r + f] * w, o[p * S::v_cols + 2 * k + 1][2 * r + f] * w);
          if constexpr (S::v_words == 4) *reinterpret_cast<uint4*>(out + d) = make_uint4(v[0], v[1], v[2], v[3]);
          else if constexpr (S::v_words == 2) *reinterpret_cast<uint2*>(out + d) = make_uint2(v[0], v[1]);
          else *reinterpret_cast<uint32_t*>(out + d) = v[0];
        }
      if (a.lse != nullptr && t == 0) a.lse[h * q_rows + (long long)seq * a.rq.T + i] = l[r] > 0.f ? m[r] + log2f(l[r]) : CUDART_INF_F;
    }
    return;
  }
  if (t == 0)
#pragma unroll
    for (int r = 0; r < 2; ++r) { s_m[warp][g + 8 * r] = m[r]; s_l[warp][g + 8 * r] = l[r]; }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    float all = kNone;
    for (int w = 0; w < kWarps; ++w) all = fmaxf(all, s_m[w][g + 8 * r]);
    const float by = m[r] == kNone ? 0.f : ex2(m[r] - all);
#pragma unroll
    for (int p = 0; p < S::v_pieces; ++p)
#pragma unroll
      for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int i = 0; i < S::v_cols; ++i) s_o[warp][g + 8 * r][(p * 8 + 2 * t + f) * S::v_cols + i] = o[p * S::v_cols + i][2 * r + f] * by;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < kRowsM * kD / 2; e += 32 * kWarps) {
    const int r = e / (kD / 2), d = e % (kD / 2) * 2, row = row0 + r;
    if (row >= rows || d >= a.D) continue;
    float all = kNone, sum = 0.f, x = 0.f, y = 0.f;
    for (int w = 0; w < kWarps; ++w) all = fmaxf(all, s_m[w][r]);
    for (int w = 0; w < kWarps; ++w) {
      sum += s_m[w][r] == kNone ? 0.f : s_l[w][r] * ex2(s_m[w][r] - all);
      x += s_o[w][r][d];
      y += s_o[w][r][d + 1];
    }
    if (plan.splits > 1) {
      const long long at_part = (unit * plan.splits + blockIdx.y) * kRowsM + r;
      *reinterpret_cast<float2*>(part + at_part * kD + d) = make_float2(x, y);
      if (d == 0) {
        part_ml[2 * at_part] = all;
        part_ml[2 * at_part + 1] = sum;
      }
      continue;
    }
    const int i = row / R, h = kh * R + row % R;
    const float w = sum > 0.f ? 1.f / sum : 0.f;
    *reinterpret_cast<uint32_t*>(at_out(a.o, seq, i, h) + d) = pack_bf16(x * w, y * w);
    if (a.lse != nullptr && d == 0) a.lse[h * q_rows + (long long)seq * a.rq.T + i] = sum > 0.f ? all + log2f(sum) : CUDART_INF_F;
  }
}

// Splits of one row, in order.  A block of kD / 2 threads per row.
template <int kD>
__global__ void __launch_bounds__(kD / 2) attention_few_join_kernel(const __grid_constant__ AttnArgs a, const FewPlan plan, const float* __restrict__ part,
                                                                    const float* __restrict__ part_ml) {
  pdl_sync();
  const int R = a.H / a.G, rows = a.rq.T * R;
  const long long unit = blockIdx.x / kRowsM;
  const int r = blockIdx.x % kRowsM, row = (int)(unit % plan.row_blocks) * kRowsM + r, d = threadIdx.x * 2;
  if (row >= rows || d >= a.D) return;
  const int kh = (int)(unit / plan.row_blocks % a.G), seq = (int)(unit / plan.row_blocks / a.G);
  const long long first = unit * plan.splits * kRowsM + r;
  float all = kNone, sum = 0.f, x = 0.f, y = 0.f;
  for (int s = 0; s < plan.splits; ++s) all = fmaxf(all, part_ml[2 * (first + (long long)s * kRowsM)]);
  for (int s = 0; s < plan.splits; ++s) {
    const long long at_part = first + (long long)s * kRowsM;
    const float m = part_ml[2 * at_part];
    const float by = m == kNone ? 0.f : ex2(m - all);
    if (by == 0.f) continue;
    const float2 v = *reinterpret_cast<const float2*>(part + at_part * kD + d);
    sum += part_ml[2 * at_part + 1] * by;
    x += v.x * by;
    y += v.y * by;
  }
  const int i = row / R, h = kh * R + row % R;
  const float w = sum > 0.f ? 1.f / sum : 0.f;
  *reinterpret_cast<uint32_t*>(at_out(a.o, seq, i, h) + d) = pack_bf16(x * w, y * w);
  if (a.lse != nullptr && d == 0) a.lse[h * ((long long)a.B * a.rq.T) + (long long)seq * a.rq.T + i] = sum > 0.f ? all + log2f(sum) : CUDART_INF_F;
}

int few_columns(const AttnArgs& a) { return a.D <= 16 ? 16 : a.D <= 32 ? 32 : a.D <= 64 ? 64 : 128; }

FewPlan plan_of(const AttnArgs& a) {
  FewPlan p{};
  p.row_blocks = (int)(((long long)a.rq.T * (a.H / a.G) + kRowsM - 1) / kRowsM);
  const long long units = (long long)a.B * a.G * p.row_blocks;
  const int keys = a.rk.T;
  p.per_unit = keys <= 256 && units >= 148 * 8 ? 1 : kWarps;
  p.splits = 1;
  p.chunk = keys;
  if (p.per_unit > 1) {
    const long long want = (148 * 4 + units - 1) / units;           // blocks that fill the GPU
    const long long most = (keys + 255) / 256;
    long long s = want < most ? want : most;
    if (s < (keys + 1023) / 1024 && a.rk.len != nullptr) s = (keys + 1023) / 1024;      // lengths may be anything: long ones are shared
    if (s > 1024) s = 1024;
    p.chunk = (int)((keys + s - 1) / s + 63) / 64 * 64;
    p.splits = (keys + p.chunk - 1) / p.chunk;
  }
  return p;
}

template <int kD>
cudaError_t launch(const AttnArgs& a, const FewPlan& p, float* work, cudaStream_t st) {
  const long long units = (long long)a.B * a.G * p.row_blocks;
  float* ml = work == nullptr ? nullptr : work + units * p.splits * kRowsM * kD;
  const long long blocks = p.per_unit == 1 ? (units + kWarps - 1) / kWarps : units;
  if (units * kRowsM >= (1LL << 31)) return cudaErrorInvalidConfiguration;
  cudaError_t e = launch_pdl(attention_few_kernel<kD>, dim3((unsigned)blocks, p.splits), dim3(32 * kWarps), 0, st, a, p, work, ml);
  if (e != cudaSuccess || p.splits == 1) return e;
  return launch_pdl(attention_few_join_kernel<kD>, dim3((unsigned)(units * kRowsM)), dim3(kD / 2), 0, st, a, p, (const float*)work, (const float*)ml);
}

}  // namespace

bool attention_few_takes(const AttnArgs& a) { return a.rq.off == nullptr && (long long)a.rq.T * (a.H / a.G) <= 4 * kRowsM; }

long long attention_few_floats(const AttnArgs& a) {
  const FewPlan p = plan_of(a);
  return p.splits == 1 ? 0 : (long long)a.B * a.G * p.row_blocks * p.splits * kRowsM * (few_columns(a) + 2);
}

const char* launch_attention_few(const AttnArgs& a, float* work, cudaStream_t st) {
  const FewPlan p = plan_of(a);
  const int D = few_columns(a);
  cudaError_t e = D == 16 ? launch<16>(a, p, work, st) : D == 32 ? launch<32>(a, p, work, st) : D == 64 ? launch<64>(a, p, work, st) : launch<128>(a, p, work, st);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

}  // namespace tn
