// Layer normalisation of rows, forward and backward.
//
//   mean = sum x / C,  var = sum (x - mean)^2 / C,  r = 1 / sqrt(var + eps),  xh = (x - mean) r
//   y = xh gamma + beta
//   dx = r (g - mean(g) - xh mean(g xh))  with g = dy gamma;  dgamma = sum over rows of dy xh;  dbeta = sum over rows of dy
//
// One pass over the data each way: a row lies in the registers of a group of threads (a power of two of them, up to a block of 512),
// so the variance is summed around the mean that was just found, without reading x again.  Sums are fp32.  Rows of more than 8192
// elements (of some widths from 8186 on, as they start anywhere in 16 bytes) are read again for each sum, by a block of 1024 and out of L2.
// What bounds it is memory where rows are within a warp: x once and y once forward, x and dy once and dx once backward.  Measured, fp32
// 409600 x 64: 39 us forward (5.4 TB/s), 62 us backward (5.0 TB/s), its sums over rows included.  Rows that a block shares wait twice
// for its sum of two numbers, and with 16 elements per thread the instructions between the waits take longer than the loads: bf16
// 8192 x 6413 72 us forward (2.9 TB/s), 107 us backward (2.9 TB/s).
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
#include "attention_tc.cuh"
#include "tn_ops.h"

namespace tn {

namespace {

constexpr int kBlock = 256;          // threads of a block whose groups are a warp or less
constexpr int kPerThread = 16;       // elements of a row that a thread holds, at most
// Within a warp, groups double before threads hold more than these: 409600 fp32 rows of 64 take 38.9 us forward and 62.4 us
// backward so, 39.0 us and 70.6 us with twice the elements (fewer registers, more warps with loads under way), 8192 rows of
// 429 14.4 and 21.6 against 14.4 and 23.5, 200 bf16 rows of 64 6.2 us against 8.2 us.
constexpr int kPerLane = 8;
constexpr int kWideBlock = 512;

template <typename T> struct Piece;
template <> struct Piece<float> {
  static constexpr int n = 4;
  __device__ __forceinline__ static void unpack(const uint4& v, float* f) {
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
  __device__ __forceinline__ static void unpack(const uint4& v, float* f) {
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
  __device__ __forceinline__ static void unpack(const uint4& v, float* f) {
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

// Sum over the tpr threads of a group in a warp
template <int kN>
__device__ __forceinline__ void warp_sum(float (&v)[kN], int tpr) {
#pragma unroll
  for (int i = 0; i < kN; ++i)
    for (int o = tpr / 2; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
}

// Sum over the block.  `s`: two rows of 32 times kN values that take turns, so that one barrier per sum is enough.
template <int kN>
__device__ __forceinline__ void block_sum(float (&v)[kN], int threads, float2* s, int& turn) {
  warp_sum<kN>(v, 32);
  float* row = reinterpret_cast<float*>(s) + turn * 32 * kN;
  turn ^= 1;
  const int warp = threadIdx.x >> 5, warps = threads >> 5;      // an even number
  if ((threadIdx.x & 31) == 0)
#pragma unroll
    for (int i = 0; i < kN; ++i) row[warp * kN + i] = v[i];
  __syncthreads();
  float2 sum = make_float2(0.f, 0.f);
  for (int w = 0; w < warps * kN / 2; ++w) sum = attn::add2(sum, *reinterpret_cast<const float2*>(row + 2 * w));
  if (kN == 1) v[0] = sum.x + sum.y;
  else { v[0] = sum.x; v[kN - 1] = sum.y; }
}

// Columns of a piece that lie in the row: the piece's first element is column `c0` (negative in front of the row).
__device__ __forceinline__ bool in_row(int c, int C) { return (unsigned)c < (unsigned)C; }

// A thread's piece number p of a row: all of it lies in the row, or only some elements do.
template <int n>
__device__ __forceinline__ bool whole_piece(int p, int shift, int C) { return p * n >= shift && p * n + n <= shift + C; }
template <int n>
__device__ __forceinline__ void keep_row(float2 (&f)[n / 2], int p, int shift, int C) {
#pragma unroll
  for (int e = 0; e < n / 2; ++e) {
    if (!in_row(p * n + 2 * e - shift, C)) f[e].x = 0.f;
    if (!in_row(p * n + 2 * e + 1 - shift, C)) f[e].y = 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void pairs_of(const uint4& v, float2* f) { Piece<T>::unpack(v, reinterpret_cast<float*>(f)); }

// kNV pieces per thread, 32 / tpr rows or more per warp
template <typename T, int kNV>
__global__ void __launch_bounds__(kBlock)
layer_norm_fwd_kernel(const T* __restrict__ x, const float* __restrict__ gamma, const float* __restrict__ beta, float eps, long long rows, int C,
                      int tpr, T* __restrict__ y, float* __restrict__ stats) {
  constexpr int n = Piece<T>::n;
  using namespace attn;
  pdl_sync();
  const int t = threadIdx.x % tpr;
  const int per_block = blockDim.x / tpr;
  const long long groups = (long long)gridDim.x * per_block;
  const long long first = (long long)blockIdx.x * per_block + threadIdx.x / tpr;
  const int shift = (int)((first * C) % n);            // the same for all rows of the group
  const long long total = rows * C, step = groups * C / n;
  const float inv = 1.f / (float)C;

  float2 g[kNV][n / 2], b[kNV][n / 2];
#pragma unroll
  for (int i = 0; i < kNV; ++i)
#pragma unroll
    for (int e = 0; e < n; ++e) {
      const int c = (t + i * tpr) * n + e - shift;
      reinterpret_cast<float*>(g[i])[e] = gamma != nullptr && in_row(c, C) ? gamma[c] : 1.f;
      reinterpret_cast<float*>(b[i])[e] = beta != nullptr && in_row(c, C) ? beta[c] : 0.f;
    }
  const int pieces = (shift + C + n - 1) / n;
  long long at = (first * C - shift) / n + t;           // of the thread's first piece
  uint4 v[kNV];
  auto fetch = [&](long long from) {
#pragma unroll
    for (int i = 0; i < kNV; ++i)
      if (t + i * tpr < pieces) v[i] = load_piece(x, from + i * tpr, total);
  };
  // Threads of one warp may belong to rows on both sides of the end; all of them take part in the sums.
  if (first < rows) fetch(at);
  for (long long r = first, lead = first - (threadIdx.x % 32) / tpr; lead < rows; r += groups, lead += groups, at += step) {
    float2 f[kNV][n / 2], m2 = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kNV; ++i) {
      pairs_of<T>(v[i], f[i]);
      if (!whole_piece<n>(t + i * tpr, shift, C)) keep_row<n>(f[i], t + i * tpr, shift, C);
#pragma unroll
      for (int e = 0; e < n / 2; ++e) m2 = add2(m2, f[i][e]);
    }
    if (r + groups < rows) fetch(at + step);           // in flight beside the sums
    float m[1] = {m2.x + m2.y};
    warp_sum<1>(m, tpr);
    const float mean = m[0] * inv;
    float2 q2 = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kNV; ++i) {
#pragma unroll
      for (int e = 0; e < n / 2; ++e) f[i][e] = add2(f[i][e], both(-mean));
      if (!whole_piece<n>(t + i * tpr, shift, C)) keep_row<n>(f[i], t + i * tpr, shift, C);
#pragma unroll
      for (int e = 0; e < n / 2; ++e) q2 = fma2(f[i][e], f[i][e], q2);
    }
    float q[1] = {q2.x + q2.y};
    warp_sum<1>(q, tpr);
    const float rstd = 1.f / sqrtf(q[0] * inv + eps);
    if (r >= rows) continue;
#pragma unroll
    for (int i = 0; i < kNV; ++i) {
      const int p = t + i * tpr;
      if (p >= pieces) continue;
#pragma unroll
      for (int e = 0; e < n / 2; ++e) f[i][e] = fma2(mul2(f[i][e], both(rstd)), g[i][e], b[i][e]);
      store_piece(y, at + i * tpr, reinterpret_cast<const float*>(f[i]), shift - p * n, shift + C - p * n);
    }
    if (stats != nullptr && t == 0) {
      stats[r] = mean;
      stats[rows + r] = rstd;
    }
  }
}

// part: [gridDim.x][2][C], the block's sums of dgamma and dbeta; null where they are not wanted
template <typename T, int kNV>
__global__ void __launch_bounds__(kBlock)
layer_norm_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x, const float* __restrict__ stats, const float* __restrict__ gamma,
                      long long rows, int C, int tpr, T* __restrict__ dx, float* __restrict__ part) {
  constexpr int n = Piece<T>::n;
  using namespace attn;
  pdl_sync();
  extern __shared__ float s_part[];                      // [groups of the block][2][C]
  const int t = threadIdx.x % tpr;
  const int per_block = blockDim.x / tpr;
  const int group = threadIdx.x / tpr;
  const long long groups = (long long)gridDim.x * per_block;
  const long long first = (long long)blockIdx.x * per_block + group;
  const int shift = (int)((first * C) % n);
  const long long total = rows * C, step = groups * C / n;
  const float inv = 1.f / (float)C;

  float2 g[kNV][n / 2], sg[kNV][n / 2], sb[kNV][n / 2];
#pragma unroll
  for (int i = 0; i < kNV; ++i) {
#pragma unroll
    for (int e = 0; e < n; ++e) {
      const int c = (t + i * tpr) * n + e - shift;
      reinterpret_cast<float*>(g[i])[e] = gamma != nullptr && in_row(c, C) ? gamma[c] : 1.f;
    }
#pragma unroll
    for (int e = 0; e < n / 2; ++e) sg[i][e] = sb[i][e] = make_float2(0.f, 0.f);
  }
  const int pieces = (shift + C + n - 1) / n;
  long long at = (first * C - shift) / n + t;
  uint4 vx[kNV], vd[kNV];
  float mean_next = 0.f, rstd_next = 0.f;
  auto fetch = [&](long long r, long long from) {
    mean_next = stats[r];
    rstd_next = stats[rows + r];
#pragma unroll
    for (int i = 0; i < kNV; ++i)
      if (t + i * tpr < pieces) {
        vx[i] = load_piece(x, from + i * tpr, total);
        vd[i] = load_piece(dy, from + i * tpr, total);
      }
  };
  if (first < rows) fetch(first, at);
  for (long long r = first, lead = first - (threadIdx.x % 32) / tpr; lead < rows; r += groups, lead += groups, at += step) {
    const bool there = r < rows;
    const float mean = mean_next, rstd = rstd_next;
    float2 fx[kNV][n / 2], fd[kNV][n / 2], m0 = make_float2(0.f, 0.f), m1 = m0;
#pragma unroll
    for (int i = 0; i < kNV; ++i) {
      pairs_of<T>(vx[i], fx[i]);
      pairs_of<T>(vd[i], fd[i]);
#pragma unroll
      for (int e = 0; e < n / 2; ++e) fx[i][e] = mul2(add2(fx[i][e], both(-mean)), both(rstd));
      if (!there || !whole_piece<n>(t + i * tpr, shift, C)) {
        keep_row<n>(fx[i], t + i * tpr, shift, there ? C : 0);
        keep_row<n>(fd[i], t + i * tpr, shift, there ? C : 0);
      }
#pragma unroll
      for (int e = 0; e < n / 2; ++e) {
        sb[i][e] = add2(sb[i][e], fd[i][e]);
        sg[i][e] = fma2(fd[i][e], fx[i][e], sg[i][e]);
        fd[i][e] = mul2(fd[i][e], g[i][e]);
        m0 = add2(m0, fd[i][e]);
        m1 = fma2(fd[i][e], fx[i][e], m1);
      }
    }
    if (r + groups < rows) fetch(r + groups, at + step);
    if (dx == nullptr) continue;
    float m[2] = {m0.x + m0.y, m1.x + m1.y};
    warp_sum<2>(m, tpr);
    if (!there) continue;
    const float c1 = m[0] * inv, c2 = m[1] * inv;
#pragma unroll
    for (int i = 0; i < kNV; ++i) {
      const int p = t + i * tpr;
      if (p >= pieces) continue;
#pragma unroll
      for (int e = 0; e < n / 2; ++e) fd[i][e] = mul2(fma2(fx[i][e], both(-c2), add2(fd[i][e], both(-c1))), both(rstd));
      store_piece(dx, at + i * tpr, reinterpret_cast<const float*>(fd[i]), shift - p * n, shift + C - p * n);
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
      float* to = s_part + (size_t)group * 2 * C;
      to[c] = reinterpret_cast<const float*>(sg[i])[e];
      to[C + c] = reinterpret_cast<const float*>(sb[i])[e];
    }
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

// ---- rows that a block shares: through a ring in shared memory --------------------------------------------------------------------
// A block's sums have barriers in between, and what hides them is rows on their way: one lane asks for rows ahead with bulk copies, of
// the 16-byte pieces that a row lies in.  Gain and shift lie in shared memory too, moved by the rows' shift.
constexpr int kRing = 3;

__device__ __forceinline__ void row_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// Where the rows of a block lie.  The last piece of the tensor may be cut short: it is read by itself (tail).
template <typename T>
struct RowSpan {
  static constexpr int n = Piece<T>::n;
  long long total;
  int C, shift, pieces;
  __device__ __forceinline__ long long first_piece(long long r) const { return (r * C - shift) / n; }
  __device__ __forceinline__ int whole_pieces(long long r) const {
    const long long left = total / n - first_piece(r);
    return left < pieces ? (int)left : pieces;
  }
};

template <typename T>
__global__ void __launch_bounds__(kWideBlock, 2)
layer_norm_row_fwd_kernel(const T* __restrict__ x, const float* __restrict__ gamma, const float* __restrict__ beta, float eps, long long rows, int C,
                          int slot_bytes, T* __restrict__ y, float* __restrict__ stats, int* status) {
  constexpr int n = Piece<T>::n, kNV = kPerThread / n;      // (with half as many per thread, half the threads would hold the row)
  using namespace attn;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ __align__(8) uint64_t s_full[kRing];
  __shared__ float2 s_sum[32];
  __shared__ int s_abort_i;
  const int t = threadIdx.x, tpr = blockDim.x;
  if (t == 0) {
    for (int s = 0; s < kRing; ++s) tc::mbar_init(tc::smem_u32(&s_full[s]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    s_abort_i = 0;
  }
  __syncthreads();
  pdl_sync();
  RowSpan<T> span{rows * C, C, (int)(((long long)blockIdx.x * C) % n), 0};
  span.pieces = (span.shift + C + n - 1) / n;
  const int shift = span.shift, pieces = span.pieces, pad = pieces * n;
  float* s_g = reinterpret_cast<float*>(smem + kRing * slot_bytes);
  float* s_b = s_g + pad;
  const uint32_t ring = tc::smem_u32(smem);
  // four elements of each piece, then the other four: neighbouring threads read neighbouring 16 bytes
  auto place = [&](int i) { return (i % n / 4 * pieces + i / n) * 4 + i % 4; };
  auto ask = [&](long long r, int s) {
    const uint32_t bytes = span.whole_pieces(r) * 16, bar = tc::smem_u32(&s_full[s]);
    tc::mbar_expect_tx(bar, bytes);
    if (bytes) row_copy(ring + s * slot_bytes, reinterpret_cast<const uint4*>(x) + span.first_piece(r), bytes, bar);
  };
  if (t == 0)
    for (int s = 0; s < kRing; ++s)
      if (blockIdx.x + (long long)s * gridDim.x < rows) ask(blockIdx.x + (long long)s * gridDim.x, s);
  for (int i = t; i < pad; i += tpr) {
    const bool in = in_row(i - shift, C);
    s_g[place(i)] = in && gamma != nullptr ? gamma[i - shift] : 1.f;
    s_b[place(i)] = in && beta != nullptr ? beta[i - shift] : 0.f;
  }
  __syncthreads();
  const float inv = 1.f / (float)C;
  int turn = 0, s = 0, phase = 0;
  bool ok = true;
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    ok = ok && tc::mbar_wait(tc::smem_u32(&s_full[s]), phase, &s_abort_i);
    if (!ok) s_abort_i = 1;      // (the block's barriers are passed all the same)
    const int whole = span.whole_pieces(r);
    float2 f[kNV][n / 2], m2 = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kNV; ++i) {
      const int p = t + i * tpr;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (p < whole) v = *reinterpret_cast<const uint4*>(smem + s * slot_bytes + p * 16);
      else if (p < pieces) v = load_piece(x, span.first_piece(r) + p, span.total);
      pairs_of<T>(v, f[i]);
      if (!whole_piece<n>(p, shift, C)) keep_row<n>(f[i], p, shift, C);
#pragma unroll
      for (int e = 0; e < n / 2; ++e) m2 = add2(m2, f[i][e]);
    }
    float m[1] = {m2.x + m2.y};
    block_sum<1>(m, tpr, s_sum, turn);
    // behind the barrier nobody reads the slot any more
    if (t == 0 && r + (long long)kRing * gridDim.x < rows) ask(r + (long long)kRing * gridDim.x, s);
    const float mean = m[0] * inv;
    float2 q2 = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kNV; ++i) {
      const int p = t + i * tpr;
#pragma unroll
      for (int e = 0; e < n / 2; ++e) f[i][e] = add2(f[i][e], both(-mean));
      if (!whole_piece<n>(p, shift, C)) keep_row<n>(f[i], p, shift, C);
#pragma unroll
      for (int e = 0; e < n / 2; ++e) q2 = fma2(f[i][e], f[i][e], q2);
    }
    float q[1] = {q2.x + q2.y};
    block_sum<1>(q, tpr, s_sum, turn);
    const float rstd = 1.f / sqrtf(q[0] * inv + eps);
    const long long at = span.first_piece(r);
#pragma unroll
    for (int i = 0; i < kNV; ++i) {
      const int p = t + i * tpr;
      if (p < pieces) {
#pragma unroll
        for (int e = 0; e < n / 2; e += 2) {
          const float4 g = *reinterpret_cast<const float4*>(s_g + (e / 2 * pieces + p) * 4), b = *reinterpret_cast<const float4*>(s_b + (e / 2 * pieces + p) * 4);
          f[i][e] = fma2(mul2(f[i][e], both(rstd)), make_float2(g.x, g.y), make_float2(b.x, b.y));
          f[i][e + 1] = fma2(mul2(f[i][e + 1], both(rstd)), make_float2(g.z, g.w), make_float2(b.z, b.w));
        }
        store_piece(y, at + p, reinterpret_cast<const float*>(f[i]), shift - p * n, shift + C - p * n);
      }
    }
    if (stats != nullptr && t == 0) {
      stats[r] = mean;
      stats[rows + r] = rstd;
    }
    if (++s == kRing) { s = 0; phase ^= 1; }
  }
  __syncthreads();
  if (s_abort_i) {
    if (t == 0) set_status(status, kMbarTimeout, 44, (int)blockIdx.x);
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);        // copies in flight land
  }
}

template <typename T>
__global__ void __launch_bounds__(kWideBlock)
layer_norm_row_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x, const float* __restrict__ stats, const float* __restrict__ gamma,
                          long long rows, int C, int slot_bytes, T* __restrict__ dx, float* __restrict__ part, int* status) {
  constexpr int n = Piece<T>::n, kNV = kPerThread / n;      // (with half as many per thread, half the threads would hold the row)
  using namespace attn;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ __align__(8) uint64_t s_full[kRing];
  __shared__ float2 s_sum[64];
  __shared__ int s_abort_i;
  const int t = threadIdx.x, tpr = blockDim.x;
  if (t == 0) {
    for (int s = 0; s < kRing; ++s) tc::mbar_init(tc::smem_u32(&s_full[s]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    s_abort_i = 0;
  }
  __syncthreads();
  pdl_sync();
  RowSpan<T> span{rows * C, C, (int)(((long long)blockIdx.x * C) % n), 0};
  span.pieces = (span.shift + C + n - 1) / n;
  const int shift = span.shift, pieces = span.pieces, pad = pieces * n;
  float* s_g = reinterpret_cast<float*>(smem + 2 * kRing * slot_bytes);
  const uint32_t ring = tc::smem_u32(smem);
  // four elements of each piece, then the other four: neighbouring threads read neighbouring 16 bytes
  auto place = [&](int i) { return (i % n / 4 * pieces + i / n) * 4 + i % 4; };
  auto ask = [&](long long r, int s) {
    const uint32_t bytes = span.whole_pieces(r) * 16, bar = tc::smem_u32(&s_full[s]);
    tc::mbar_expect_tx(bar, 2 * bytes);
    if (bytes) {
      row_copy(ring + 2 * s * slot_bytes, reinterpret_cast<const uint4*>(x) + span.first_piece(r), bytes, bar);
      row_copy(ring + (2 * s + 1) * slot_bytes, reinterpret_cast<const uint4*>(dy) + span.first_piece(r), bytes, bar);
    }
  };
  if (t == 0)
    for (int s = 0; s < kRing; ++s)
      if (blockIdx.x + (long long)s * gridDim.x < rows) ask(blockIdx.x + (long long)s * gridDim.x, s);
  for (int i = t; i < pad; i += tpr) s_g[place(i)] = gamma != nullptr && in_row(i - shift, C) ? gamma[i - shift] : 1.f;
  __syncthreads();
  const float inv = 1.f / (float)C;
  float2 sg[kNV][n / 2], sb[kNV][n / 2];
#pragma unroll
  for (int i = 0; i < kNV; ++i)
#pragma unroll
    for (int e = 0; e < n / 2; ++e) sg[i][e] = sb[i][e] = make_float2(0.f, 0.f);
  int turn = 0, s = 0, phase = 0;
  bool ok = true;
  float mean_next = 0.f, rstd_next = 0.f;
  if (blockIdx.x < rows) { mean_next = stats[blockIdx.x]; rstd_next = stats[rows + blockIdx.x]; }
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const float mean = mean_next, rstd = rstd_next;
    if (r + gridDim.x < rows) { mean_next = stats[r + gridDim.x]; rstd_next = stats[rows + r + gridDim.x]; }
    ok = ok && tc::mbar_wait(tc::smem_u32(&s_full[s]), phase, &s_abort_i);
    if (!ok) s_abort_i = 1;
    const int whole = span.whole_pieces(r);
    uint4 vx[kNV], vd[kNV];
    float2 m0 = make_float2(0.f, 0.f), m1 = m0;
    auto gain = [&](int p, float2 (&g)[n / 2]) {
#pragma unroll
      for (int e = 0; e < n / 2; e += 2) {
        const float4 v = *reinterpret_cast<const float4*>(s_g + (e / 2 * pieces + p) * 4);
        g[e] = make_float2(v.x, v.y);
        g[e + 1] = make_float2(v.z, v.w);
      }
    };
#pragma unroll
    for (int i = 0; i < kNV; ++i) {
      const int p = t + i * tpr;
      if (p >= pieces) continue;
      if (p < whole) {
        vx[i] = *reinterpret_cast<const uint4*>(smem + 2 * s * slot_bytes + p * 16);
        vd[i] = *reinterpret_cast<const uint4*>(smem + (2 * s + 1) * slot_bytes + p * 16);
      } else {
        vx[i] = load_piece(x, span.first_piece(r) + p, span.total);
        vd[i] = load_piece(dy, span.first_piece(r) + p, span.total);
      }
      float2 fx[n / 2], fd[n / 2], g[n / 2];
      pairs_of<T>(vx[i], fx);
      pairs_of<T>(vd[i], fd);
      gain(p, g);
#pragma unroll
      for (int e = 0; e < n / 2; ++e) fx[e] = mul2(add2(fx[e], both(-mean)), both(rstd));
      if (!whole_piece<n>(p, shift, C)) {
        keep_row<n>(fx, p, shift, C);
        keep_row<n>(fd, p, shift, C);
      }
#pragma unroll
      for (int e = 0; e < n / 2; ++e) {
        sb[i][e] = add2(sb[i][e], fd[e]);
        sg[i][e] = fma2(fd[e], fx[e], sg[i][e]);
        fd[e] = mul2(fd[e], g[e]);
        m0 = add2(m0, fd[e]);
        m1 = fma2(fd[e], fx[e], m1);
      }
    }
    float m[2] = {m0.x + m0.y, m1.x + m1.y};
    block_sum<2>(m, tpr, s_sum, turn);
    if (t == 0 && r + (long long)kRing * gridDim.x < rows) ask(r + (long long)kRing * gridDim.x, s);
    const float c1 = m[0] * inv, c2 = m[1] * inv;
    const long long at = span.first_piece(r);
    if (dx != nullptr)
#pragma unroll
      for (int i = 0; i < kNV; ++i) {
        const int p = t + i * tpr;
        if (p >= pieces) continue;
        float2 fx[n / 2], fd[n / 2], g[n / 2];
        pairs_of<T>(vx[i], fx);
        pairs_of<T>(vd[i], fd);
        gain(p, g);
#pragma unroll
        for (int e = 0; e < n / 2; ++e) {
          fx[e] = mul2(add2(fx[e], both(-mean)), both(rstd));
          fd[e] = mul2(fma2(fx[e], both(-c2), fma2(fd[e], g[e], both(-c1))), both(rstd));
        }
        store_piece(dx, at + p, reinterpret_cast<const float*>(fd), shift - p * n, shift + C - p * n);
      }
    if (++s == kRing) { s = 0; phase ^= 1; }
  }
  if (part != nullptr) {
    float* out = part + (size_t)blockIdx.x * 2 * C;
#pragma unroll
    for (int i = 0; i < kNV; ++i)
#pragma unroll
      for (int e = 0; e < n; ++e) {
        const int c = (t + i * tpr) * n + e - shift;
        if (in_row(c, C)) {
          out[c] = reinterpret_cast<const float*>(sg[i])[e];
          out[C + c] = reinterpret_cast<const float*>(sb[i])[e];
        }
      }
  }
  __syncthreads();
  if (s_abort_i) {
    if (t == 0) set_status(status, kMbarTimeout, 45, (int)blockIdx.x);
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);        // copies in flight land
  }
}

// ---- rows too wide for the registers of a block: read again for each sum, out of L2 ----------------------------------------------
template <typename T>
__global__ void __launch_bounds__(1024) layer_norm_wide_fwd_kernel(const T* __restrict__ x, const float* __restrict__ gamma,
                                                                   const float* __restrict__ beta, float eps, long long rows, int C,
                                                                   T* __restrict__ y, float* __restrict__ stats) {
  pdl_sync();
  __shared__ float2 s_sum[32];
  int turn = 0;
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* row = x + r * C;
    float m[1] = {0.f};
    for (int c = threadIdx.x; c < C; c += 1024) m[0] += Piece<T>::get(row[c]);
    block_sum<1>(m, 1024, s_sum, turn);
    const float mean = m[0] / (float)C;
    float q[1] = {0.f};
    for (int c = threadIdx.x; c < C; c += 1024) {
      const float d = Piece<T>::get(row[c]) - mean;
      q[0] += d * d;
    }
    block_sum<1>(q, 1024, s_sum, turn);
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
  __shared__ float2 s_sum[64];
  int turn = 0;
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const float mean = stats[r], rstd = stats[rows + r];
    float m[2] = {0.f, 0.f};
    for (int c = threadIdx.x; c < C; c += 1024) {
      const float d = Piece<T>::get(dy[r * C + c]) * (gamma ? gamma[c] : 1.f);
      m[0] += d;
      m[1] += d * (Piece<T>::get(x[r * C + c]) - mean) * rstd;
    }
    block_sum<2>(m, 1024, s_sum, turn);
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
  while (p.tpr * ((p.tpr < 32 ? kPerLane : kPerThread) / n) < need && p.tpr < kWideBlock) p.tpr <<= 1;
  p.wide = p.tpr * (kPerThread / n) < need;
  p.nv = 1;
  while (p.tpr * p.nv < need && p.nv < kPerThread / n) p.nv <<= 1;
  p.block = p.tpr > 32 ? p.tpr : kBlock;
  p.per_block = p.tpr > 32 ? 1 : kBlock / p.tpr;
  p.blocks = (rows + p.per_block - 1) / p.per_block;
  return p;
}

// The bytes of a row in the ring, wherever it starts in a piece.
template <typename T>
int slot_bytes(int C) { return (C + 2 * (Piece<T>::n - 1)) / Piece<T>::n * 16; }

// As many blocks as fit on the GPU at a time, a multiple of eight: rows of a group then start at one place in a 16-byte piece.
template <typename K>
int resident_grid(K kernel, int block, size_t smem, long long blocks) {
  struct Fit { const void* kernel; int dev, block, all; size_t smem; };      // what the driver has said before
  thread_local Fit known[16] = {};
  thread_local int next = 0;
  int dev = 0, all = 0;
  cudaGetDevice(&dev);
  for (const Fit& f : known)
    if (f.kernel == (const void*)kernel && f.dev == dev && f.block == block && f.smem == smem) all = f.all;
  if (all == 0) {
    int sms = 148, per_sm = 1;
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, block, smem) != cudaSuccess || per_sm < 1) per_sm = 1;
    all = sms * per_sm;
    known[next] = {(const void*)kernel, dev, block, all, smem};
    next = (next + 1) % 16;
  }
  long long g = all / 8 * 8;
  if (blocks < g) g = (blocks + 7) / 8 * 8;
  return (int)(g < 8 ? 8 : g);
}

template <typename T, typename F>
const char* with_pieces(const Plan& p, F&& f) {
  constexpr int most = kPerThread / Piece<T>::n;
  if (p.nv == 1) return f(std::integral_constant<int, 1>{});
  if (p.nv == 2) return f(std::integral_constant<int, 2>{});
  return f(std::integral_constant<int, most>{});
}

const char* told(cudaError_t e) {
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

// Rows of the workspace where a row is too wide for a block's registers
int wide_sum_rows(long long rows) { return rows < 64 ? (int)rows : 64; }

template <typename T>
const char* fwd(const LayerNormArgs& a, cudaStream_t st) {
  const Plan p = plan_of<T>(a.rows, a.C);
  if (p.wide) {
    const int grid = (int)(a.rows < 592 ? a.rows : 592);
    return told(launch_pdl(layer_norm_wide_fwd_kernel<T>, dim3(grid), dim3(1024), 0, st, (const T*)a.x, a.gamma, a.beta, a.eps, a.rows, a.C,
                           (T*)a.y, a.stats));
  }
  return with_pieces<T>(p, [&](auto nv) -> const char* {
    constexpr int kNV = decltype(nv)::value;
    if (p.tpr <= 32) {
      auto* k = layer_norm_fwd_kernel<T, kNV>;
      return told(launch_pdl(k, dim3(resident_grid(k, p.block, 0, p.blocks)), dim3(p.block), 0, st, (const T*)a.x, a.gamma, a.beta, a.eps, a.rows,
                             a.C, p.tpr, (T*)a.y, a.stats));
    }
    auto* k = layer_norm_row_fwd_kernel<T>;
    const int slot = slot_bytes<T>(a.C);
    const size_t smem = kRing * slot + 2 * slot / sizeof(T) * sizeof(float);
    cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);      // of the current device
    return told(launch_pdl(k, dim3(resident_grid(k, p.block, smem, p.blocks)), dim3(p.block), smem, st, (const T*)a.x, a.gamma, a.beta, a.eps,
                           a.rows, a.C, slot, (T*)a.y, a.stats, a.status));
  });
}

template <typename T>
const char* bwd(const LayerNormArgs& a, int* part_rows, cudaStream_t st) {
  const Plan p = plan_of<T>(a.rows, a.C);
  const bool sums = a.dgamma != nullptr || a.dbeta != nullptr;
  if (p.wide) {
    const int shares = wide_sum_rows(a.rows);
    if (part_rows) { *part_rows = shares; return nullptr; }
    const int grid = (int)(a.rows < 592 ? a.rows : 592);
    if (a.dx != nullptr)
      if (const char* err = told(launch_pdl(layer_norm_wide_bwd_kernel<T>, dim3(grid), dim3(1024), 0, st, (const T*)a.dy, (const T*)a.x, a.stats,
                                            a.gamma, a.rows, a.C, (T*)a.dx)))
        return err;
    if (sums) {
      if (const char* err = told(launch_pdl(layer_norm_wide_sums_kernel<T>, dim3((a.C + 127) / 128, shares), dim3(128), 0, st,
                                            (const T*)a.dy, (const T*)a.x, a.stats, a.rows, a.C, a.part)))
        return err;
      return told(launch_pdl(layer_norm_add_kernel, dim3((unsigned)((2LL * a.C + 31) / 32)), dim3(32 * kAddRows), 0, st, a.part, shares, a.C, a.dgamma,
                             a.dbeta));
    }
    return nullptr;
  }
  return with_pieces<T>(p, [&](auto nv) -> const char* {
    constexpr int kNV = decltype(nv)::value;
    int grid;
    const char* err = nullptr;
    if (p.tpr <= 32) {
      auto* k = layer_norm_bwd_kernel<T, kNV>;
      const size_t smem = (size_t)p.per_block * 2 * a.C * sizeof(float);      // at most 32 KiB: a thread has 16 elements
      grid = resident_grid(k, p.block, smem, p.blocks);
      if (!part_rows)
        err = told(launch_pdl(k, dim3(grid), dim3(p.block), smem, st, (const T*)a.dy, (const T*)a.x, a.stats, a.gamma, a.rows, a.C, p.tpr, (T*)a.dx,
                              sums ? a.part : nullptr));
    } else {
      auto* k = layer_norm_row_bwd_kernel<T>;
      const int slot = slot_bytes<T>(a.C);
      const size_t smem = 2 * kRing * slot + slot / sizeof(T) * sizeof(float);
      cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);      // of the current device
      grid = resident_grid(k, p.block, smem, p.blocks);
      if (!part_rows)
        err = told(launch_pdl(k, dim3(grid), dim3(p.block), smem, st, (const T*)a.dy, (const T*)a.x, a.stats, a.gamma, a.rows, a.C, slot, (T*)a.dx,
                              sums ? a.part : nullptr, a.status));
    }
    if (part_rows) { *part_rows = grid; return nullptr; }
    if (err || !sums) return err;
    return told(launch_pdl(layer_norm_add_kernel, dim3((unsigned)((2LL * a.C + 31) / 32)), dim3(32 * kAddRows), 0, st, a.part, grid, a.C, a.dgamma, a.dbeta));
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
