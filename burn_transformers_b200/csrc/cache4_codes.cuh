// Codes of the 4-bit cache (cache4.cuh) as bfloat16 values, two at a time.
//
// A code n becomes the bfloat16 128 + n by setting the exponent's bits over it; (128 + n) s - 136 s, one multiply-add, is the value
// (n - 8) s exactly: 136 s = 17 s 2^3 has 8 significant bits, and the value has 7.
#pragma once
#include "common.cuh"

namespace bt {

// Nibble I of both halves of `w`, as 128 + n.
template <int I>
__device__ __forceinline__ unsigned c4_pair(unsigned w) {
  return ((w >> (4 * I)) & 0x000f000fu) | 0x43004300u;
}
__device__ __forceinline__ unsigned c4_fma2(unsigned a, unsigned b, unsigned c) {
  unsigned d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;\n" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
// A scale byte's bfloat16 bits (low half): 2^((b >> 3) - 20) (1 + (b & 7) / 8), or NaN.
__device__ __forceinline__ unsigned c4_scale_bits(unsigned b) { return b == 255u ? 0x7fc0u : b * 16u + 0x3580u; }
// -136 s of two scales.
__device__ __forceinline__ unsigned c4_shift(unsigned s2) { return c4_fma2(s2, 0xc308c308u, 0x80008000u); }

}  // namespace bt
