// Instructions and layouts that the tensor-core attention kernels share.
//
// Every operand tile lies in shared memory as chunks of 64 columns, [rows][128 bytes] with the 128-byte swizzle, so that one tile
// serves as either side of a product: along its columns (K-major) for q k^T, along its rows (MN-major) for p v.
#pragma once
#include <cuda.h>
#include <type_traits>
#include "attention_rows.cuh"
#include "tc_primitives.cuh"

namespace tn {
namespace attn {

using namespace tc;

constexpr float kNone = -__builtin_huge_valf();

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Two fp32 operations in one instruction
__device__ __forceinline__ unsigned long long bits_of(float2 a) { return *reinterpret_cast<unsigned long long*>(&a); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(bits_of(a)), "l"(bits_of(b)), "l"(bits_of(c)));
  return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  unsigned long long d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits_of(a)), "l"(bits_of(b)));
  return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits_of(a)), "l"(bits_of(b)));
  return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 both(float a) { return make_float2(a, a); }

// 2^x for two at a time without the special function unit, which makes 16 a cycle and SM: x = n + f, a polynomial for 2^f on
// [-1/2, 1/2] (least squares reweighted towards the smallest largest relative error: 2.7e-6 in fp32), n added to the exponent.  What
// comes of -125 is taken off in the end, so that all below, minus infinity too, comes as zero.
__device__ __forceinline__ float2 ex2_poly(float2 x) {
  constexpr float c0 = 0.9999992847442627f;
  x = make_float2(fmaxf(x.x, -125.f), fmaxf(x.y, -125.f));
  const float2 r = add2(x, both(12582912.f));                     // 1.5 2^23: the integer is in the low bits
  const float2 f = fma2(add2(r, both(-12582912.f)), both(-1.f), x);
  float2 p = fma2(f, both(0.009570101276040077f), both(0.05591785907745361f));
  p = fma2(f, p, both(0.240247443318367f));
  p = fma2(f, p, both(0.6931217908859253f));
  p = fma2(f, p, both(c0));
  p.x = __int_as_float(__float_as_int(p.x) + (__float_as_int(r.x) << 23));
  p.y = __int_as_float(__float_as_int(p.y) + (__float_as_int(r.y) << 23));
  return add2(p, both(-c0 * 2.3509887016445750e-38f));           // 2^-125
}

// tanh for |y| <= 1: y times a polynomial in y^2, least squares reweighted towards the smallest largest relative error (5.9e-7, 7.0e-7 in
// fp32): with a cap far above it, a score has to be off by little of its own size.  No exponential, and two at a time.
__device__ __forceinline__ float2 tanh_small(float2 y) {
  const float2 z = mul2(y, y);
  float2 p = fma2(z, both(-0.0030670601408928633f), both(0.016743114218115807f));
  p = fma2(z, p, both(-0.051605671644210815f));
  p = fma2(z, p, both(0.13281433284282684f));
  p = fma2(z, p, both(-0.3332904279232025f));
  p = fma2(z, p, both(0.9999994039535522f));
  return mul2(y, p);
}
// and for any y.  1 - 2 / (1 + e^2y), one exponential, is off by some 2^-22 of 1, which may be all of a small tanh: a score is off by that
// much of its cap.  Up to kCoarseCap that is 2^-14, little beside the 2^-8 that rounding to bf16 moves its weight by; above, small values come
// of the polynomial, each by itself, in instances of their own: 8192 causal tokens x 16 heads x 128 columns 487 + 1074 us in place of 404 +
// 1050, 4096 sequences of 1 to 200 x 4 heads x 16 columns 127 + 300 in place of 119 + 288.
constexpr float kCoarseCap = 256.f;
enum Cap { kUncapped, kCapped, kCappedFar };
template <Cap kCap>
__device__ __forceinline__ float2 tanh_any(float2 y) {
  const float2 far = make_float2(1.f - __fdividef(2.f, 1.f + ex2(2.f * kLog2e * y.x)), 1.f - __fdividef(2.f, 1.f + ex2(2.f * kLog2e * y.y)));
  if (kCap != kCappedFar) return far;
  const float2 near = tanh_small(y);
  return make_float2(fabsf(y.x) <= 1.f ? near.x : far.x, fabsf(y.y) <= 1.f ? near.y : far.y);
}
// launch(...) of the instance that a call wants
template <typename F>
cudaError_t with_cap(const AttnArgs& a, F&& launch) {
  if (!(a.cap > 0.f)) return launch(std::integral_constant<Cap, kUncapped>{});
  if (a.cap <= kCoarseCap) return launch(std::integral_constant<Cap, kCapped>{});
  return launch(std::integral_constant<Cap, kCappedFar>{});
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int t, int h, int b, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(t), "r"(h), "r"(b)
      : "memory");
}
// A from tensor memory: lane = row, two bf16 along the contraction per column
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accum)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]), "r"(r[1]),
      "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
      "r"(r[14]), "r"(r[15]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
template <int kCols>
__device__ __forceinline__ uint32_t tmem_alloc(uint32_t* slot) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "n"(kCols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  return 0;
}
template <int kCols>
__device__ __forceinline__ void tmem_dealloc(uint32_t tmem) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kCols) : "memory");
}

// fp32 results of bf16 operands, 128 rows, n columns; b_mn: B lies with its output columns behind one another
__device__ __forceinline__ uint32_t idesc_of(int n, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}
// What a descriptor grows by for step s of 16: along the columns of a tile of kRows rows (K-major), along its rows (MN-major)
template <int kRows>
__device__ constexpr uint64_t step_k(int s) { return (uint64_t)(((s >> 2) * (kRows * 128) + (s & 3) * 32) >> 4); }
__device__ constexpr uint64_t step_mn(int s) { return (uint64_t)((s * 2048) >> 4); }

// `v`, the same for all lanes, in a form that the compiler knows to be: descriptors and coordinates made of it need not be collected
// from a lane's registers for each instruction
__device__ __forceinline__ int one_of_warp(int v) { return __shfl_sync(0xffffffffu, v, 0); }

__device__ __forceinline__ int round16(int n) { return (n + 15) & ~15; }

// Rows [from, to) of a tile set to zero by one warp: rows behind the end of a sequence hold anything, and a weight of zero times a
// NaN is a NaN.
template <int kRows>
__device__ __forceinline__ void zero_rows(uint8_t* tile, int chunks, int from, int to, int lane) {
  const int per = (to - from) * 8;
  for (int i = lane; i < per * chunks; i += 32)
    *reinterpret_cast<uint4*>(tile + (i / per) * (kRows * 128) + from * 128 + (i % per) * 16) = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  __syncwarp();
}

// Eight bf16 of zero, or of fp32 values times w, to a row
__device__ __forceinline__ uint4 pack8(const float* f, float w) {
  return make_uint4(pack_bf16(f[0] * w, f[1] * w), pack_bf16(f[2] * w, f[3] * w), pack_bf16(f[4] * w, f[5] * w), pack_bf16(f[6] * w, f[7] * w));
}

// What is left of eight fp32 values times w when pack8 has rounded them
__device__ __forceinline__ uint4 rest8(const float* f, float w, const uint4& r) {
  const uint32_t v[4] = {r.x, r.y, r.z, r.w};
  float d[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    d[2 * i] = f[2 * i] * w - __uint_as_float(v[i] << 16);
    d[2 * i + 1] = f[2 * i + 1] * w - __uint_as_float(v[i] & 0xffff0000u);
  }
  return pack8(d, 1.f);
}

// [rows, 64 columns] boxes of an operand; columns beyond D and rows beyond T come as zeros
bool operand_map(const AttnOperand& o, int D, const AttnRows& r, int B, int heads, int box_rows, CUtensorMap* out);

}  // namespace attn
}  // namespace tn
