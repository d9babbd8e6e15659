// The 4-bit latent record, 416 bytes a token: two halves of 208, one for each CTA of the pair that attends over it.  Half c:
//   128 bytes  codes of the latent values 256 c .. 256 c + 255, eight to a 32-bit word
//    16 bytes  the scales of their sixteen groups of 16 values
//    64 bytes  rope values 32 c .. 32 c + 31, bf16
// A scale byte (e << 3) + m stands for (8 + m) 2^(e - 18), 255 for NaN.  A code is a sign and the number of one of 0, .5, 1, 1.5, 2, 3, 4, 6
// (two bits of exponent, one of mantissa).  Value = code x scale: two and four significant bits, exact in bf16.
// Word: even values in the low 16 bits, odd ones in the high 16; of the four in a half, value k has its sign and number at bits
//   k = 0: 15, 8 7 6     k = 1: 12, 5 4 3     k = 2: 9, 2 1 0     k = 3: 14, 11 10 13
// so that a pair of values becomes a pair of bf16 -- sign at 15, number at 8 7 6, which is where the two low exponent bits and the top
// mantissa bit are: the code times 2^-126 -- by a shift and a mask, k = 3 by three.  With codes side by side each pair takes two of either.
#pragma once
#include <stdint.h>

namespace dsa {

constexpr int kLatent4Bytes = 416, kLatent4Half = 208, kLatent4Scales = 128, kLatent4Rope = 144;      // offsets within a half
constexpr uint32_t kLatent4Nan = 255;

__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// Eight codes of a word as bf16 pairs (values 2k, 2k + 1 in r[k]), times 2^-126.
__device__ __forceinline__ void latent4_codes(uint32_t w, uint32_t (&r)[4]) {
  constexpr uint32_t kM = 0x81c081c0u;
  r[0] = w & kM;
  r[1] = (w << 3) & kM;
  r[2] = (w << 6) & kM;
  r[3] = ((w << 1) & 0x80008000u) | ((w >> 3) & 0x01800180u) | ((w >> 7) & 0x00400040u);
}
// A scale byte as a pair of bf16, times 2^112: the byte's exponent field moved by 224, so that 255 becomes a NaN.
__device__ __forceinline__ uint32_t latent4_scale(uint32_t byte) { return byte * 0x00100010u + 0x70007000u; }
// So code x scale comes out times this: q's latent values are taken times its inverse, and the output too.
constexpr float kLatent4Gain = 16384.f;                // 2^14
constexpr uint32_t kLatent4GainPair = 0x46804680u;     // the same as a pair of bf16

}  // namespace dsa
