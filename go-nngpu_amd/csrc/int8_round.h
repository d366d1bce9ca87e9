// int8_round.h — the arithmetic of a quantised row, shared by the kernels that quantise.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace gn {

// The scale of a row from the bits of its largest magnitude (ordered as the values are, infinity and NaN above all numbers).
__device__ __forceinline__ float int8_scale(uint32_t top) {
  return top >= 0x7f800000u ? NAN : fmaxf(__uint_as_float(top) / 127.0f, 0x1p-126f);
}

// y / s rounded to the nearest integer, ties to the even one, of the exact quotient: k from an approximate quotient is off by one at
// most, and only where the quotient is next to a middle. r = y - k s is exact there: for |y| >= s both terms are multiples of
// s's last place and |r| is below s; below that k is 0, or 1 where r is exact or at least not rounded past s / 2.
// inv: about 1 / s. The result is a float.
__device__ __forceinline__ float int8_round(float y, float s, float inv) {
  float k = rintf(y * inv);
  const float r = fmaf(-k, s, y), a = fabsf(r), half = 0.5f * s;
  if (a >= half) {  // seldom: whole waves skip it
    const bool odd = fabsf(k - 2.0f * rintf(0.5f * k)) == 1.0f;
    if (a > half || odd) k += copysignf(1.0f, r);
  }
  return k;
}

// Four of them as bytes: 1.5 2^23 + k has k's two's complement in its low bits.
__device__ __forceinline__ uint32_t int8_pack(float a, float b, float c, float d) {
  constexpr float kMagic = 12582912.0f;
  const uint32_t ab = __builtin_amdgcn_perm(__float_as_uint(b + kMagic), __float_as_uint(a + kMagic), 0x0c0c0400);
  const uint32_t cd = __builtin_amdgcn_perm(__float_as_uint(d + kMagic), __float_as_uint(c + kMagic), 0x04000c0c);
  return ab | cd;
}

// A value as it is in fp32. Without this the compiler may take a product and its conversion to fp16 as one instruction, which
// rounds once where the definition rounds twice.
__device__ __forceinline__ float as_fp32(float x) {
  asm("" : "+v"(x));
  return x;
}

}  // namespace gn
