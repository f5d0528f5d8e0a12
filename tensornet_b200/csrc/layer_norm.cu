// Layer normalisation of rows, forward and backward.
//
//   mean = sum x / C,  var = sum (x - mean)^2 / C,  r = 1 / sqrt(var + eps),  xh = (x - mean) r
//   y = xh gamma + beta
//   dx = r (g - mean(g) - xh mean(g xh))  with g = dy gamma;  dgamma = sum over rows of dy xh;  dbeta = sum over rows of dy
//
// One pass over the data each way: a row lies in the registers of a group of threads (a power of two of them, up to a block of
// 512), so the variance is summed around the mean that was just found, without reading x again.  Sums are fp32.
// What bounds it is memory: x once and y once forward, x and dy once and dx once backward.
//
// Rows of any width are read in 16-byte pieces.  Where the width is no multiple of a piece, rows start anywhere in one; a piece
// then belongs to two rows, each of which takes its own elements of it.  A group takes every G-th row, G a multiple of the
// elements of a piece, so all its rows start at the same place in a piece and its threads see the same columns each time: gain
// and shift, and the sums of their gradients, stay in registers for all rows of a group.
// The sums of a block are added in shared memory and written to a row of a workspace, and a second kernel adds the rows of the
// workspace: every order is fixed, so results are the same each time.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <type_traits>
#include "tn_device.cuh"
#include "tn_ops.h"

namespace tn {

namespace {

constexpr int kBlock = 256;          // threads of a block whose groups are a warp or less
constexpr int kPerThread = 16;       // elements of a row that a thread holds
constexpr int kWideBlock = 512;

template <typename T> struct Piece;
template <> struct Piece<float> {
  static constexpr int n = 4;
  __device__ static void unpack(const uint4& v, float* f) {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
  }
  __device__ static uint4 pack(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
  __device__ static float get(float v) { return v; }
  __device__ static float put(float v) { return v; }
};
template <> struct Piece<__nv_bfloat16> {
  static constexpr int n = 8;
  __device__ static void unpack(const uint4& v, float* f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  __device__ static uint4 pack(const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ static float get(__nv_bfloat16 v) { return __bfloat162float(v); }
  __device__ static __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};
template <> struct Piece<__half> {
  static constexpr int n = 8;
  __device__ static void unpack(const uint4& v, float* f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  }
  __device__ static uint4 pack(const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ static float get(__half v) { return __half2float(v); }
  __device__ static __half put(float v) { return __float2half_rn(v); }
};

// The piece `at` (in pieces from the start of the tensor, which lies on 16 bytes).  Only the tensor's last one can be cut short.
template <typename T>
__device__ __forceinline__ uint4 load_piece(const T* p, long long at, long long total) {
  constexpr int n = Piece<T>::n;
  if ((at + 1) * n <= total) return __ldg(reinterpret_cast<const uint4*>(p) + at);
  __align__(16) T part[n];
#pragma unroll
  for (int e = 0; e < n; ++e) part[e] = at * n + e < total ? p[at * n + e] : Piece<T>::put(0.f);
  return *reinterpret_cast<const uint4*>(part);
}

// Elements [lo, hi) of a piece
template <typename T>
__device__ __forceinline__ void store_piece(T* p, long long at, const float* f, int lo, int hi) {
  constexpr int n = Piece<T>::n;
  if (lo <= 0 && hi >= n) {
    reinterpret_cast<uint4*>(p)[at] = Piece<T>::pack(f);
    return;
  }
#pragma unroll
  for (int e = 0; e < n; ++e)
    if (e >= lo && e < hi) p[at * n + e] = Piece<T>::put(f[e]);
}

// Sum over the threads of a group: part of a warp, or the block.  `s`: two rows of 32 floats that take turns, so that one barrier
// per sum is enough.
template <bool kBlockRow, int kN>
__device__ __forceinline__ void group_sum(float (&v)[kN], int tpr, float* s, int& turn) {
#pragma unroll
  for (int i = 0; i < kN; ++i)
    for (int o = (kBlockRow ? 16 : tpr / 2); o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  if (!kBlockRow) return;
  float* row = s + turn * 32 * kN;
  turn ^= 1;
  const int warp = threadIdx.x >> 5, warps = tpr >> 5;
  if ((threadIdx.x & 31) == 0)
#pragma unroll
    for (int i = 0; i < kN; ++i) row[warp * kN + i] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kN; ++i) v[i] = 0.f;
  for (int w = 0; w < warps; ++w)
#pragma unroll
    for (int i = 0; i < kN; ++i) v[i] += row[w * kN + i];
}

// Columns of a piece that lie in the row: the piece's first element is column `c0` (negative in front of the row).
__device__ __forceinline__ bool in_row(int c, int C) { return (unsigned)c < (unsigned)C; }

// kNV pieces per thread; kBlockRow: a row per block, else 32 / tpr rows or more per warp.
template <typename T, int kNV, bool kBlockRow>
__global__ void __launch_bounds__(kBlockRow ? kWideBlock : kBlock)
layer_norm_fwd_kernel(const T* __restrict__ x, const float* __restrict__ gamma, const float* __restrict__ beta, float eps, long long rows, int C,
                      int tpr, T* __restrict__ y, float* __restrict__ stats) {
  constexpr int n = Piece<T>::n;
  pdl_sync();
  __shared__ float s_sum[64];
  int turn = 0;
  const int t = kBlockRow ? threadIdx.x : threadIdx.x % tpr;
  const int per_block = kBlockRow ? 1 : blockDim.x / tpr;
  const long long groups = (long long)gridDim.x * per_block;
  const long long first = (long long)blockIdx.x * per_block + (kBlockRow ? 0 : threadIdx.x / tpr);
  const int shift = (int)((first * C) % n);            // the same for all rows of the group
  const long long total = rows * C;
  const float inv = 1.f / (float)C;

  float g[kNV * n], b[kNV * n];
#pragma unroll
  for (int i = 0; i < kNV; ++i)
#pragma unroll
    for (int e = 0; e < n; ++e) {
      const int c = (t + i * tpr) * n + e - shift;
      g[i * n + e] = gamma != nullptr && in_row(c, C) ? gamma[c] : 1.f;
      b[i * n + e] = beta != nullptr && in_row(c, C) ? beta[c] : 0.f;
    }
  const int pieces = (shift + C + n - 1) / n;
  uint4 v[kNV];
  auto fetch = [&](long long r) {
    const long long at = (r * C - shift) / n;
#pragma unroll
    for (int i = 0; i < kNV; ++i)
      if (t + i * tpr < pieces) v[i] = load_piece(x, at + t + i * tpr, total);
  };
  // Threads of one warp may belong to rows on both sides of the end; all of them take part in the sums.
  const long long last = kBlockRow ? rows : first - (kBlockRow ? 0 : (threadIdx.x % 32) / tpr);
  if (first < rows) fetch(first);
  for (long long r = first, lead = last; kBlockRow ? r < rows : lead < rows; r += groups, lead += groups) {
    float f[kNV * n];
    float m[1] = {0.f};
#pragma unroll
    for (int i = 0; i < kNV; ++i) {
      Piece<T>::unpack(v[i], f + i * n);
#pragma unroll
      for (int e = 0; e < n; ++e) {
        if (!in_row((t + i * tpr) * n + e - shift, C)) f[i * n + e] = 0.f;
        m[0] += f[i * n + e];
      }
    }
    if (r + groups < rows) fetch(r + groups);           // in flight beside the sums
    group_sum<kBlockRow, 1>(m, tpr, s_sum, turn);
    const float mean = m[0] * inv;
    float q[1] = {0.f};
#pragma unroll
    for (int i = 0; i < kNV; ++i)
#pragma unroll
      for (int e = 0; e < n; ++e) {
        const float d = f[i * n + e] - mean;
        f[i * n + e] = d;
        if (in_row((t + i * tpr) * n + e - shift, C)) q[0] += d * d;
      }
    group_sum<kBlockRow, 1>(q, tpr, s_sum, turn);
    const float rstd = 1.f / sqrtf(q[0] * inv + eps);
    if (r >= rows) continue;
    const long long at = (r * C - shift) / n;
#pragma unroll
    for (int i = 0; i < kNV; ++i) {
      const int p = t + i * tpr;
      if (p >= pieces) continue;
      float o[n];
#pragma unroll
      for (int e = 0; e < n; ++e) o[e] = f[i * n + e] * rstd * g[i * n + e] + b[i * n + e];
      store_piece(y, at + p, o, shift - p * n, shift + C - p * n);
    }
    if (stats != nullptr && t == 0) {
      stats[r] = mean;
      stats[rows + r] = rstd;
    }
  }
}

// part: [gridDim.x][2][C], the block's sums of dgamma and dbeta; null where they are not wanted
template <typename T, int kNV, bool kBlockRow>
__global__ void __launch_bounds__(kBlockRow ? kWideBlock : kBlock)
layer_norm_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x, const float* __restrict__ stats, const float* __restrict__ gamma,
                      long long rows, int C, int tpr, T* __restrict__ dx, float* __restrict__ part) {
  constexpr int n = Piece<T>::n;
  pdl_sync();
  __shared__ float s_sum[128];
  extern __shared__ float s_part[];                      // [groups of the block][2][C]
  int turn = 0;
  const int t = kBlockRow ? threadIdx.x : threadIdx.x % tpr;
  const int per_block = kBlockRow ? 1 : blockDim.x / tpr;
  const int group = kBlockRow ? 0 : threadIdx.x / tpr;
  const long long groups = (long long)gridDim.x * per_block;
  const long long first = (long long)blockIdx.x * per_block + group;
  const int shift = (int)((first * C) % n);
  const long long total = rows * C;
  const float inv = 1.f / (float)C;

  float g[kNV * n], sg[kNV * n], sb[kNV * n];
#pragma unroll
  for (int i = 0; i < kNV; ++i)
#pragma unroll
    for (int e = 0; e < n; ++e) {
      const int c = (t + i * tpr) * n + e - shift;
      g[i * n + e] = gamma != nullptr && in_row(c, C) ? gamma[c] : 1.f;
      sg[i * n + e] = sb[i * n + e] = 0.f;
    }
  const int pieces = (shift + C + n - 1) / n;
  uint4 vx[kNV], vd[kNV];
  float mean_next = 0.f, rstd_next = 0.f;
  auto fetch = [&](long long r) {
    const long long at = (r * C - shift) / n;
    mean_next = stats[r];
    rstd_next = stats[rows + r];
#pragma unroll
    for (int i = 0; i < kNV; ++i)
      if (t + i * tpr < pieces) {
        vx[i] = load_piece(x, at + t + i * tpr, total);
        vd[i] = load_piece(dy, at + t + i * tpr, total);
      }
  };
  const long long lead0 = kBlockRow ? first : first - (threadIdx.x % 32) / tpr;
  if (first < rows) fetch(first);
  for (long long r = first, lead = lead0; lead < rows; r += groups, lead += groups) {
    const bool there = r < rows;
    const float mean = mean_next, rstd = rstd_next;
    float fx[kNV * n], fd[kNV * n];
    float m[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kNV; ++i) {
      Piece<T>::unpack(vx[i], fx + i * n);
      Piece<T>::unpack(vd[i], fd + i * n);
#pragma unroll
      for (int e = 0; e < n; ++e) {
        const int k = i * n + e;
        const bool in = there && in_row((t + i * tpr) * n + e - shift, C);
        fx[k] = in ? (fx[k] - mean) * rstd : 0.f;
        fd[k] = in ? fd[k] : 0.f;
        sb[k] += fd[k];
        sg[k] += fd[k] * fx[k];
        fd[k] *= g[k];
        m[0] += fd[k];
        m[1] += fd[k] * fx[k];
      }
    }
    if (r + groups < rows) fetch(r + groups);
    if (dx == nullptr) continue;
    group_sum<kBlockRow, 2>(m, tpr, s_sum, turn);
    if (!there) continue;
    const float c1 = m[0] * inv, c2 = m[1] * inv;
    const long long at = (r * C - shift) / n;
#pragma unroll
    for (int i = 0; i < kNV; ++i) {
      const int p = t + i * tpr;
      if (p >= pieces) continue;
      float o[n];
#pragma unroll
      for (int e = 0; e < n; ++e) o[e] = rstd * (fd[i * n + e] - c1 - fx[i * n + e] * c2);
      store_piece(dx, at + p, o, shift - p * n, shift + C - p * n);
    }
  }
  if (part == nullptr) return;
  float* out = part + (size_t)blockIdx.x * 2 * C;
#pragma unroll
  for (int i = 0; i < kNV; ++i)
#pragma unroll
    for (int e = 0; e < n; ++e) {
      const int c = (t + i * tpr) * n + e - shift;
      if (!in_row(c, C)) continue;
      float* to = kBlockRow ? out : s_part + (size_t)group * 2 * C;
      to[c] = sg[i * n + e];
      to[C + c] = sb[i * n + e];
    }
  if (kBlockRow) return;
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * C; c += blockDim.x) {
    float s = 0.f;
    for (int k = 0; k < per_block; ++k) s += s_part[(size_t)k * 2 * C + c];
    out[c] = s;
  }
}

// out[c] = sum over `n` of part[n][columns]; the first C columns go to `a`, the others to `b` (either may be null)
constexpr int kAddRows = 16;
__global__ void __launch_bounds__(32 * kAddRows) layer_norm_add_kernel(const float* __restrict__ part, int n, int C, float* a, float* b) {
  pdl_sync();
  __shared__ double s[kAddRows][32];
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5;
  const long long c = (long long)blockIdx.x * 32 + lane;
  double v = 0.0;
  if (c < 2LL * C)
    for (int k = row; k < n; k += kAddRows) v += (double)part[(size_t)k * 2 * C + c];
  s[row][lane] = v;
  __syncthreads();
  if (row != 0 || c >= 2LL * C) return;
  for (int k = 1; k < kAddRows; ++k) v += s[k][lane];
  float* to = c < C ? a : b;
  if (to != nullptr) to[c < C ? c : c - C] = (float)v;
}

// ---- rows too wide for the registers of a block: read again for each sum, out of L2 ----------------------------------------------
template <typename T>
__global__ void __launch_bounds__(1024) layer_norm_wide_fwd_kernel(const T* __restrict__ x, const float* __restrict__ gamma,
                                                                   const float* __restrict__ beta, float eps, long long rows, int C,
                                                                   T* __restrict__ y, float* __restrict__ stats) {
  pdl_sync();
  __shared__ float s_sum[64];
  int turn = 0;
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* row = x + r * C;
    float m[1] = {0.f};
    for (int c = threadIdx.x; c < C; c += 1024) m[0] += Piece<T>::get(row[c]);
    group_sum<true, 1>(m, 1024, s_sum, turn);
    const float mean = m[0] / (float)C;
    float q[1] = {0.f};
    for (int c = threadIdx.x; c < C; c += 1024) {
      const float d = Piece<T>::get(row[c]) - mean;
      q[0] += d * d;
    }
    group_sum<true, 1>(q, 1024, s_sum, turn);
    const float rstd = 1.f / sqrtf(q[0] / (float)C + eps);
    for (int c = threadIdx.x; c < C; c += 1024) {
      const float v = (Piece<T>::get(row[c]) - mean) * rstd;
      y[r * C + c] = Piece<T>::put(v * (gamma ? gamma[c] : 1.f) + (beta ? beta[c] : 0.f));
    }
    if (stats != nullptr && threadIdx.x == 0) {
      stats[r] = mean;
      stats[rows + r] = rstd;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(1024) layer_norm_wide_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                                   const float* __restrict__ stats, const float* __restrict__ gamma,
                                                                   long long rows, int C, T* __restrict__ dx) {
  pdl_sync();
  __shared__ float s_sum[128];
  int turn = 0;
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const float mean = stats[r], rstd = stats[rows + r];
    float m[2] = {0.f, 0.f};
    for (int c = threadIdx.x; c < C; c += 1024) {
      const float d = Piece<T>::get(dy[r * C + c]) * (gamma ? gamma[c] : 1.f);
      m[0] += d;
      m[1] += d * (Piece<T>::get(x[r * C + c]) - mean) * rstd;
    }
    group_sum<true, 2>(m, 1024, s_sum, turn);
    const float c1 = m[0] / (float)C, c2 = m[1] / (float)C;
    for (int c = threadIdx.x; c < C; c += 1024) {
      const float d = Piece<T>::get(dy[r * C + c]) * (gamma ? gamma[c] : 1.f);
      dx[r * C + c] = Piece<T>::put(rstd * (d - c1 - (Piece<T>::get(x[r * C + c]) - mean) * rstd * c2));
    }
  }
}

// a block has 128 columns and every gridDim.y-th row
template <typename T>
__global__ void __launch_bounds__(128) layer_norm_wide_sums_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                                   const float* __restrict__ stats, long long rows, int C,
                                                                   float* __restrict__ part) {
  pdl_sync();
  const int c = blockIdx.x * 128 + threadIdx.x;
  if (c >= C) return;
  float sg = 0.f, sb = 0.f;
  for (long long r = blockIdx.y; r < rows; r += gridDim.y) {
    const float d = Piece<T>::get(dy[r * C + c]);
    sb += d;
    sg += d * (Piece<T>::get(x[r * C + c]) - stats[r]) * stats[rows + r];
  }
  part[(size_t)blockIdx.y * 2 * C + c] = sg;
  part[(size_t)blockIdx.y * 2 * C + C + c] = sb;
}

struct Plan {
  bool wide;
  int tpr, nv, block, per_block;
  long long blocks;      // that have a row to start with
};

template <typename T>
Plan plan_of(long long rows, int C) {
  constexpr int n = Piece<T>::n;
  Plan p{};
  const int need = (C + (C % n ? n - 1 : 0) + n - 1) / n;      // pieces of a row, wherever it starts
  p.tpr = 1;
  while (p.tpr * (kPerThread / n) < need && p.tpr < kWideBlock) p.tpr <<= 1;
  p.wide = p.tpr * (kPerThread / n) < need;
  p.nv = 1;
  while (p.tpr * p.nv < need && p.nv < kPerThread / n) p.nv <<= 1;
  p.block = p.tpr > 32 ? p.tpr : kBlock;
  p.per_block = p.tpr > 32 ? 1 : kBlock / p.tpr;
  p.blocks = (rows + p.per_block - 1) / p.per_block;
  return p;
}

// As many blocks as fit on the GPU at a time, a multiple of eight: rows of a group then start at one place in a 16-byte piece.
template <typename K>
int resident_grid(K kernel, int block, size_t smem, long long blocks) {
  int dev = 0, sms = 148, per_sm = 1;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, block, smem) != cudaSuccess || per_sm < 1) per_sm = 1;
  long long g = (long long)sms * per_sm / 8 * 8;
  if (blocks < g) g = (blocks + 7) / 8 * 8;
  return (int)(g < 8 ? 8 : g);
}

template <typename T, typename F>
const char* with_kernel(const Plan& p, F&& f) {
  constexpr int most = kPerThread / Piece<T>::n;
  if (p.tpr > 32) {
    if (p.nv == 1) return f(std::integral_constant<int, 1>{}, std::true_type{});
    if (p.nv == 2) return f(std::integral_constant<int, 2>{}, std::true_type{});
    return f(std::integral_constant<int, most>{}, std::true_type{});
  }
  if (p.nv == 1) return f(std::integral_constant<int, 1>{}, std::false_type{});
  if (p.nv == 2) return f(std::integral_constant<int, 2>{}, std::false_type{});
  return f(std::integral_constant<int, most>{}, std::false_type{});
}

const char* told(cudaError_t e) {
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

constexpr int kWideSumRows = 64;      // rows of the workspace where a row is too wide for a block's registers

template <typename T>
const char* fwd(const LayerNormArgs& a, cudaStream_t st) {
  const Plan p = plan_of<T>(a.rows, a.C);
  if (p.wide) {
    const int grid = (int)(a.rows < 592 ? a.rows : 592);
    return told(launch_pdl(layer_norm_wide_fwd_kernel<T>, dim3(grid), dim3(1024), 0, st, (const T*)a.x, a.gamma, a.beta, a.eps, a.rows, a.C,
                           (T*)a.y, a.stats));
  }
  return with_kernel<T>(p, [&](auto nv, auto block_row) {
    auto* k = layer_norm_fwd_kernel<T, decltype(nv)::value, decltype(block_row)::value>;
    return told(launch_pdl(k, dim3(resident_grid(k, p.block, 0, p.blocks)), dim3(p.block), 0, st, (const T*)a.x, a.gamma, a.beta, a.eps, a.rows,
                           a.C, p.tpr, (T*)a.y, a.stats));
  });
}

template <typename T>
const char* bwd(const LayerNormArgs& a, int* part_rows, cudaStream_t st) {
  const Plan p = plan_of<T>(a.rows, a.C);
  const bool sums = a.dgamma != nullptr || a.dbeta != nullptr;
  if (p.wide) {
    if (part_rows) { *part_rows = kWideSumRows; return nullptr; }
    const int grid = (int)(a.rows < 592 ? a.rows : 592);
    if (a.dx != nullptr)
      if (const char* err = told(launch_pdl(layer_norm_wide_bwd_kernel<T>, dim3(grid), dim3(1024), 0, st, (const T*)a.dy, (const T*)a.x, a.stats,
                                            a.gamma, a.rows, a.C, (T*)a.dx)))
        return err;
    if (sums) {
      if (const char* err = told(launch_pdl(layer_norm_wide_sums_kernel<T>, dim3((a.C + 127) / 128, kWideSumRows), dim3(128), 0, st,
                                            (const T*)a.dy, (const T*)a.x, a.stats, a.rows, a.C, a.part)))
        return err;
      return told(launch_pdl(layer_norm_add_kernel, dim3((2 * a.C + 31) / 32), dim3(32 * kAddRows), 0, st, a.part, kWideSumRows, a.C, a.dgamma,
                             a.dbeta));
    }
    return nullptr;
  }
  return with_kernel<T>(p, [&](auto nv, auto block_row) -> const char* {
    auto* k = layer_norm_bwd_kernel<T, decltype(nv)::value, decltype(block_row)::value>;
    const size_t smem = p.tpr > 32 ? 0 : (size_t)p.per_block * 2 * a.C * sizeof(float);      // at most 32 KiB: a thread has 16 elements
    const int grid = resident_grid(k, p.block, smem, p.blocks);
    if (part_rows) { *part_rows = grid; return nullptr; }
    if (const char* err = told(launch_pdl(k, dim3(grid), dim3(p.block), smem, st, (const T*)a.dy, (const T*)a.x, a.stats, a.gamma, a.rows, a.C,
                                          p.tpr, (T*)a.dx, sums ? a.part : nullptr)))
      return err;
    if (!sums) return nullptr;
    return told(launch_pdl(layer_norm_add_kernel, dim3((2 * a.C + 31) / 32), dim3(32 * kAddRows), 0, st, a.part, grid, a.C, a.dgamma, a.dbeta));
  });
}

}  // namespace

const char* launch_layer_norm_fwd(const LayerNormArgs& a, cudaStream_t st) {
  return a.kind == 0 ? fwd<float>(a, st) : a.kind == 1 ? fwd<__nv_bfloat16>(a, st) : fwd<__half>(a, st);
}
const char* launch_layer_norm_bwd(const LayerNormArgs& a, cudaStream_t st) {
  return a.kind == 0 ? bwd<float>(a, nullptr, st) : a.kind == 1 ? bwd<__nv_bfloat16>(a, nullptr, st) : bwd<__half>(a, nullptr, st);
}
int layer_norm_part_rows(const LayerNormArgs& a) {
  int n = 0;
  a.kind == 0 ? bwd<float>(a, &n, nullptr) : a.kind == 1 ? bwd<__nv_bfloat16>(a, &n, nullptr) : bwd<__half>(a, &n, nullptr);
  return n;
}

}  // namespace tn
