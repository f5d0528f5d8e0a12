// Products of 16 rows by mma.sync whose right operands come in 4- to 16-byte pieces of rows.  Of lane number 4 g + t:
//   * rows as the right operand's columns (scores): the contraction may go over the columns of the rows in any order that both sides
//     share.  The lane takes row g at column (p 4 + t) 2 kw, kw words of two columns each; words 2 i and 2 i + 1 are the operand of
//     one product.  Left operands hold the same columns of rows g and g + 8.
//   * rows as the contraction (values): the lane takes rows 2 t, 2 t + 1, 2 t + 8 and 2 t + 9 at column (p 8 + g) vc.  Words of two
//     rows, interleaved by byte permutation, are the right operands of two products; product i has columns (p 8 + n) vc + i.
#pragma once
#include "attention_tc.cuh"

namespace tn {
namespace attn {

__device__ __forceinline__ void mma16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <int kWords, typename P>
__device__ __forceinline__ void load_words(const P* p, uint32_t* w) {
  if constexpr (kWords == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else if constexpr (kWords == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x; w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}
template <int kWords>
__device__ __forceinline__ void store_words(__nv_bfloat16* p, const uint32_t* w) {
  if constexpr (kWords == 4) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  else if constexpr (kWords == 2) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  else *reinterpret_cast<uint32_t*>(p) = w[0];
}

// Two fp32 values rounded to bf16, and what that took off
__device__ __forceinline__ uint32_t rest_of(float a, float b, uint32_t r) {
  return pack_bf16(a - __uint_as_float(r << 16), b - __uint_as_float(r & 0xffff0000u));
}

// Pieces of a row of up to kD columns
template <int kD>
struct Pieces {
  static constexpr int k_words = kD == 16 ? 2 : 4, k_pieces = kD == 16 ? 1 : kD / 32;
  static constexpr int v_words = kD >= 64 ? 4 : kD / 16, v_pieces = kD >= 64 ? kD / 64 : 1;
  static constexpr int v_cols = 2 * v_words;
  static constexpr int k_all = k_pieces * k_words;      // words of a score operand
  static constexpr int products = v_pieces * v_cols;    // of 8 columns
};

// acc[i] += a * (rows as the contraction), from the words of the lane's four rows
template <int kWords>
__device__ __forceinline__ void mma_values(float (*acc)[4], const uint32_t* a, const uint32_t (*w)[kWords]) {
#pragma unroll
  for (int i = 0; i < kWords; ++i) {
    mma16(acc[2 * i], a, __byte_perm(w[0][i], w[1][i], 0x5410), __byte_perm(w[2][i], w[3][i], 0x5410));
    mma16(acc[2 * i + 1], a, __byte_perm(w[0][i], w[1][i], 0x7632), __byte_perm(w[2][i], w[3][i], 0x7632));
  }
}

}  // namespace attn
}  // namespace tn
