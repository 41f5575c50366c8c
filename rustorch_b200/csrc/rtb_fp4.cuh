// 4-bit block-scaled tensors: e2m1 codes (0, 1/2, 1, 3/2, 2, 3, 4, 6 and a sign; the
// even column in a byte's low half) with one power-of-two scale for each 32 columns
// of a row, held as the 8-bit exponent e8m0: value = code * 2^(byte - 127).  e2m1 has
// neither infinity nor NaN: a block that holds one has byte 255, which makes all of
// its values NaN, and codes 0.
#pragma once
#include "rtb_fp8.cuh"

namespace rtb {

constexpr int kFp4Block = 32;  // columns of a scale block

// The scale byte of a block whose largest magnitude has these bits: the smallest
// power of two with amax / 2^e <= 6 = 1.5 * 2^2 (read off the bits of amax), at least
// 2^-126 so that its inverse is a normal number; 2^0 for a block of zeros.
__device__ __forceinline__ uint32_t fp4_scale_byte(uint32_t bits) {
  if (bits >= 0x7F800000u) return 255u;
  const int e = (int)(bits >> 23) - 2 + ((bits & 0x7FFFFFu) > 0x400000u);
  return bits == 0 ? 127u : (uint32_t)(e < 1 ? 1 : e);
}
// 2^(127 - byte); 0 for a block that is NaN.  (Byte 254 has no normal inverse, and no
// block: the largest exponent of fp32 gives 253.)
__device__ __forceinline__ float fp4_inverse(uint32_t byte) {
  return byte == 255 ? 0.0f : e8m0_inverse(byte);
}

// Eight codes, the first in the low half of the lowest byte, to nearest even.  |v| <=
// 6 for every value of a block but a NaN's, whose codes the caller clears.
__device__ __forceinline__ uint32_t e2m1x8(const float (&v)[8], float inv) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(v[0] * inv), "f"(v[1] * inv), "f"(v[2] * inv), "f"(v[3] * inv), "f"(v[4] * inv),
        "f"(v[5] * inv), "f"(v[6] * inv), "f"(v[7] * inv));
  return r;
}

// Eight codes -> eight floats, exactly.
__device__ __forceinline__ void e2m1x8_to_float(uint32_t eight, float (&v)[8]) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(eight));
#pragma unroll
  for (int i = 0; i < 4; ++i)
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}"
        : "=f"(v[2 * i]), "=f"(v[2 * i + 1])
        : "r"(h[i]));
}

}  // namespace rtb
