// 8-bit block-scaled tensors: e4m3 values with one power-of-two scale for each
// block of 128 columns of a row (block_rows = 1) or of 128 rows (128), held as
// the 8-bit exponent e8m0: value = q * 2^(byte - 127), byte 255 = NaN.
#pragma once
#include <cstdint>

#include "../../include/rustorch_b200.h"

namespace rtb {

constexpr int kFp8Block = 128;  // columns (and rows) of a scale block

// 2^(b - 127); 2^-127 is subnormal in fp32, 255 is NaN.
__device__ __forceinline__ float e8m0_to_float(uint32_t b) {
  const uint32_t bits = b == 0 ? 0x00400000u : (b == 255 ? 0x7FC00000u : b << 23);
  return __uint_as_float(bits);
}

// The scale byte of a block whose largest finite magnitude is amax: the
// smallest power of two with amax / 2^e <= 448 = 1.75 * 2^8 (read off the bits
// of amax), at least 2^-126 so that its inverse is a normal number; 2^0 for a
// block of zeros.  A power of two scales exactly, so a value is rounded once,
// to e4m3.
__device__ __forceinline__ uint32_t e8m0_of_amax(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int e = (int)(bits >> 23) - 8 + ((bits & 0x7FFFFFu) > 0x600000u);
  return amax == 0.0f ? 127u : (uint32_t)(e < 1 ? 1 : e);
}

// 2^(127 - b) for 1 <= b <= 253 (e8m0_of_amax gives no other).
__device__ __forceinline__ float e8m0_inverse(uint32_t b) {
  return __uint_as_float((254u - b) << 23);
}

// |x| for the block maximum: infinities and NaN do not set the scale.
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.0f;
}

// Four e4m3 codes (lowest byte first), round to nearest even.  |x * inv| <=
// 448 for every finite x; an infinity becomes NaN like a NaN does, so that it
// is not lost in the checkpoint (the conversion alone would saturate it).
__device__ __forceinline__ uint32_t e4m3x4(float x0, float x1, float x2, float x3, float inv) {
  auto fix = [](float v) { return fabsf(v) <= 448.0f ? v : __int_as_float(0x7FFFFFFF); };
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(fix(x1 * inv)), "f"(fix(x0 * inv)));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(fix(x3 * inv)), "f"(fix(x2 * inv)));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}

// Two e4m3 codes (the low 16 bits) -> two floats, exactly.
__device__ __forceinline__ float2 e4m3x2_to_float2(uint32_t two) {
  uint32_t h2;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"((uint16_t)two));
  float2 f;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}"
      : "=f"(f.x), "=f"(f.y)
      : "r"(h2));
  return f;
}

__device__ __forceinline__ float4 e4m3x4_to_float4(uint32_t four) {
  const float2 a = e4m3x2_to_float2(four & 0xFFFFu), b = e4m3x2_to_float2(four >> 16);
  return make_float4(a.x, a.y, b.x, b.y);
}

}  // namespace rtb
