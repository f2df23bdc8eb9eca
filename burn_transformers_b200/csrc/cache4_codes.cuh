// Codes of the 4-bit cache (cache4.cuh) as bfloat16 values, two at a time.
//
// The usual way to widen small whole numbers: a code n becomes the bfloat16 128 + n by setting the exponent's bits over it; (128 + n) s - 136 s, one multiply-add, is the value
// (n - 8) s exactly: 136 s = 17 s 2^3 has 8 significant bits, and the value has 7.
#pragma once
#include "common.cuh"

namespace bt {

// The two constants of c4_pair, in registers that the compiler cannot see through: an operation takes one constant only, and it would
// otherwise spend two.
struct C4Bits {
  unsigned mask, base;
  __device__ __forceinline__ C4Bits() {
    asm volatile("mov.u32 %0, 0x000f000f;\n" : "=r"(mask));
    asm volatile("mov.u32 %0, 0x43004300;\n" : "=r"(base));
  }
};
// Nibble I of both halves of `w`, as 128 + n.
template <int I>
__device__ __forceinline__ unsigned c4_pair(unsigned w, const C4Bits& c) {
  unsigned d;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;\n" : "=r"(d) : "r"(w >> (4 * I)), "r"(c.mask), "r"(c.base));      // (w & mask) | base
  return d;
}
__device__ __forceinline__ unsigned c4_fma2(unsigned a, unsigned b, unsigned c) {
  unsigned d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;\n" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
// A scale byte's bfloat16 bits (low half): 2^((b >> 3) - 20) (1 + (b & 7) / 8), or NaN.
__device__ __forceinline__ unsigned c4_scale_bits(unsigned b) { return b == 255u ? 0x7fc0u : b * 16u + 0x3580u; }
// Two scale bytes (not NaN's) as a pair of bfloat16: the multiply-adds leave the integer pipe to the codes.
__device__ __forceinline__ unsigned c4_scale_pair(unsigned lo, unsigned hi) { return hi * 0x00100000u + (lo * 16u + 0x35803580u); }
__device__ __forceinline__ unsigned c4_scale_twice(unsigned b) { return b * 0x00100010u + 0x35803580u; }
// Whether a byte of `w` is 255.
__device__ __forceinline__ bool c4_has_255(unsigned w) { return ((~w - 0x01010101u) & w & 0x80808080u) != 0u; }
// -136 s of two scales.
__device__ __forceinline__ unsigned c4_shift(unsigned s2) { return c4_fma2(s2, 0xc308c308u, 0x80008000u); }

}  // namespace bt
