// Attention within sequences, backward: a warp per row.
//
//   dv = p^T do;  dp = do v^T;  ds = p (dp - sum(do o)) (1 - tanh^2) scale;  dq = ds k;  dk = ds^T q
//
// A lane scores one key (or query) of 32, then the 32 weights pass around the warp while the lanes own columns of the result.
#include <cuda_bf16.h>
#include "attention_rows.cuh"
#include "tn_device.cuh"

namespace tn {

namespace {

using namespace attn;

constexpr int kWarps = 8;
constexpr int kCols = 4;      // columns of a row per lane, 128 / 32

__device__ __forceinline__ float dot(const __nv_bfloat16* a, const float* b, int D) {
  float s = 0.f;
  for (int d = 0; d < D; d += 8) {
    const uint4 v = *reinterpret_cast<const uint4*>(a + d);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) s += __uint_as_float(w[i] << 16) * b[d + 2 * i] + __uint_as_float(w[i] & 0xffff0000u) * b[d + 2 * i + 1];
  }
  return s;
}
__device__ __forceinline__ void load_row(const __nv_bfloat16* p, float* s, int D, int lane) {
  for (int d = lane; d < D; d += 32) s[d] = __bfloat162float(p[d]);
}
__device__ __forceinline__ void add_row(const __nv_bfloat16* p, float w, float* acc, int D, int lane) {
#pragma unroll
  for (int i = 0; i < kCols; ++i)
    if (lane + 32 * i < D) acc[i] += w * __bfloat162float(p[lane + 32 * i]);
}
__device__ __forceinline__ void store_row(__nv_bfloat16* p, const float* acc, float w, int D, int lane) {
#pragma unroll
  for (int i = 0; i < kCols; ++i)
    if (lane + 32 * i < D) p[lane + 32 * i] = __float2bfloat16_rn(acc[i] * w);
}
__device__ __forceinline__ float warp_sum(float v) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct Place {
  int seq, b, t, i, nq, nk;     // i: of the row within its sequence; seq -1: in none
  Span keys, queries;
};
// The row `at` of an operand's rows, over all sequences
__device__ __forceinline__ Place place_of(const AttnArgs& a, const AttnRows& r, long long row) {
  Place p{};
  const Tile t = tile_of(r, a.B, 1, r.off == nullptr ? (int)row : 0);
  if (r.off == nullptr) {
    p.seq = t.seq; p.b = t.seq; p.t = t.first; p.i = t.first;
  } else {
    int lo = 0, hi = a.B;       // the first offset beyond the row
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (r.off[mid] <= row) lo = mid + 1; else hi = mid;
    }
    p.seq = lo >= 1 && lo <= a.B && row < r.off[a.B] ? lo - 1 : -1;
    p.b = 0; p.t = (int)row;
    if (p.seq >= 0) p.i = (int)row - span_of(r, p.seq).first;
  }
  if (p.seq >= 0) {
    p.queries = span_of(a.rq, p.seq);
    p.keys = span_of(a.rk, p.seq);
    p.nq = p.queries.n; p.nk = p.keys.n;
    if (p.i >= span_of(r, p.seq).n) p.seq = -1;
  }
  return p;
}

__global__ void __launch_bounds__(32 * kWarps) attention_dq_kernel(const AttnArgs a, long long rows) {
  pdl_sync();
  __shared__ float s_q[kWarps][128], s_g[kWarps][128];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, h = blockIdx.y;
  const long long row = (long long)blockIdx.x * kWarps + warp;
  if (row >= rows) return;
  const Place p = place_of(a, a.rq, row);
  float acc[kCols] = {};
  if (p.seq >= 0) {
    const int g = h / (a.H / a.G), lim = keys_seen(a, p.seq, p.i, p.nq, p.nk);
    const float slope2 = a.slopes ? a.slopes[h] * kLog2e : 0.f;
    load_row(at(a.q, p.b, p.t, h), s_q[warp], a.D, lane);
    load_row(at(a.go, p.b, p.t, h), s_g[warp], a.D, lane);
    __syncwarp();
    float delta = 0.f;
    for (int d = lane; d < a.D; d += 32) delta += s_g[warp][d] * __bfloat162float(at(a.o, p.b, p.t, h)[d]);
    delta = warp_sum(delta);
    if (lane == 0) a.delta[h * rows + row] = delta;
    const float lse = a.lse[h * rows + row];
    for (int j0 = 0; j0 < lim; j0 += 32) {
      const int j = j0 + lane;
      float ds = 0.f, th = 0.f;
      if (j < lim) {
        const float s = score_of(a, dot(at(a.k, p.keys.b, p.keys.first + j, g), s_q[warp], a.D), slope2, p.i + p.nk - p.nq - j, th);
        const float dp = dot(at(a.v, p.keys.b, p.keys.first + j, g), s_g[warp], a.D);
        ds = exp2f(s - lse) * (dp - delta) * (1.f - th * th) * a.scale;
      }
      const int n = min(32, lim - j0);
      for (int k = 0; k < n; ++k) add_row(at(a.k, p.keys.b, p.keys.first + j0 + k, g), __shfl_sync(0xffffffffu, ds, k), acc, a.D, lane);
    }
  }
  store_row(at_out(a.gq, p.b, p.t, h), acc, 1.f, a.D, lane);
}

__global__ void __launch_bounds__(32 * kWarps) attention_dkv_kernel(const AttnArgs a, long long rows, long long q_rows) {
  pdl_sync();
  __shared__ float s_k[kWarps][128], s_v[kWarps][128];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = blockIdx.y;
  const long long row = (long long)blockIdx.x * kWarps + warp;
  if (row >= rows) return;
  const Place p = place_of(a, a.rk, row);
  float dk[kCols] = {}, dv[kCols] = {};
  if (p.seq >= 0) {
    load_row(at(a.k, p.b, p.t, g), s_k[warp], a.D, lane);
    load_row(at(a.v, p.b, p.t, g), s_v[warp], a.D, lane);
    __syncwarp();
    const long long flat = (a.rq.off ? 0 : (long long)p.queries.b * a.rq.T) + p.queries.first;
    for (int h = g * (a.H / a.G); h < (g + 1) * (a.H / a.G); ++h) {
      const float slope2 = a.slopes ? a.slopes[h] * kLog2e : 0.f;
      for (int i0 = 0; i0 < p.nq; i0 += 32) {
        const int i = i0 + lane;
        float w = 0.f, ds = 0.f, th = 0.f;
        if (i < p.nq && p.i < keys_seen(a, p.seq, i, p.nq, p.nk)) {
          const float s = score_of(a, dot(at(a.q, p.queries.b, p.queries.first + i, h), s_k[warp], a.D), slope2, i + p.nk - p.nq - p.i, th);
          w = exp2f(s - a.lse[h * q_rows + flat + i]);
          ds = w * (dot(at(a.go, p.queries.b, p.queries.first + i, h), s_v[warp], a.D) - a.delta[h * q_rows + flat + i]) * (1.f - th * th) * a.scale;
        }
        const int n = min(32, p.nq - i0);
        for (int k = 0; k < n; ++k) {
          const float wk = __shfl_sync(0xffffffffu, w, k), dk_w = __shfl_sync(0xffffffffu, ds, k);
          if (wk == 0.f && dk_w == 0.f) continue;
          add_row(at(a.go, p.queries.b, p.queries.first + i0 + k, h), wk, dv, a.D, lane);
          add_row(at(a.q, p.queries.b, p.queries.first + i0 + k, h), dk_w, dk, a.D, lane);
        }
      }
    }
  }
  store_row(at_out(a.gk, p.b, p.t, g), dk, 1.f, a.D, lane);
  store_row(at_out(a.gv, p.b, p.t, g), dv, 1.f, a.D, lane);
}

long long rows_of(const AttnRows& r, int B) { return r.off ? r.T : (long long)B * r.T; }
const char* told(cudaError_t e) {
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

}  // namespace

const char* launch_attention_bwd(const AttnArgs& a, cudaStream_t st) {
  const long long nq = rows_of(a.rq, a.B), nk = rows_of(a.rk, a.B);
  if (const char* e = told(launch_pdl(attention_dq_kernel, dim3((unsigned)((nq + kWarps - 1) / kWarps), a.H), dim3(32 * kWarps), 0, st, a, nq)))
    return e;
  return told(launch_pdl(attention_dkv_kernel, dim3((unsigned)((nk + kWarps - 1) / kWarps), a.G), dim3(32 * kWarps), 0, st, a, nk, nq));
}

}  // namespace tn
