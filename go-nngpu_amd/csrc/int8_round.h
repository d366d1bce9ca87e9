// int8_round.h — reading a row and the arithmetic of quantising it, shared by the kernels that do.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace gn {
namespace {

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

// 16 bytes at any address that is a multiple of T's size (the hardware takes unaligned vectors).
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Unaligned16 {
  u32x4_t v;
};
// Eight values in their own type, 0 for those at or past `left`.
template <typename T>
struct Eight;
template <>
struct Eight<float> {
  u32x4_t v[2];
  __device__ __forceinline__ float operator[](int i) const { return __uint_as_float(v[i / 4][i % 4]); }
  __device__ __forceinline__ uint32_t top() const {  // the bits of the largest magnitude
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, v[i / 4][i % 4] & 0x7fffffffu);
    return m;
  }
  __device__ __forceinline__ void load(const float *p, long left) {
    if (left >= 8) {
      v[0] = reinterpret_cast<const Unaligned16<float> *>(p)[0].v;
      v[1] = reinterpret_cast<const Unaligned16<float> *>(p)[1].v;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i / 4][i % 4] = i < left ? __float_as_uint(p[i]) : 0u;
    }
  }
};
template <>
struct Eight<_Float16> {
  half8_t v;
  __device__ __forceinline__ float operator[](int i) const { return (float)v[i]; }
  __device__ __forceinline__ uint32_t top() const {  // the bits of fp16 numbers are ordered as they are, too
    const u32x4_t b = __builtin_bit_cast(u32x4_t, v) & 0x7fff7fffu;
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, max(b[i], b[i] << 16));
    return __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)(m >> 16)));
  }
  __device__ __forceinline__ void load(const _Float16 *p, long left) {
    if (left >= 8) {
      v = __builtin_bit_cast(half8_t, reinterpret_cast<const Unaligned16<_Float16> *>(p)->v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i < left ? p[i] : (_Float16)0.0f;
    }
  }
};

// The scale of a row from the bits of its largest magnitude (ordered as the values are, infinity and NaN above all numbers).
__device__ __forceinline__ float int8_scale(uint32_t top) {
  return top >= 0x7f800000u ? NAN : fmaxf(__uint_as_float(top) / 127.0f, 0x1p-126f);
}

// y / s rounded to the nearest integer, ties to the even one, of the exact quotient, for eight values, as bytes. k from an approximate
// quotient is off by one at most, and only where the quotient is next to a middle. r = y - k s is exact there: for |y| >= s
// both terms are multiples of s's last place and |r| is below s; below that k is 0, or 1 where r is exact or at least not
// rounded past s / 2. r stands on the middle where 2 |r| = s: doubling is exact, and s / 2 is not for every s below 2^-125.
// inv: about 1 / s.
__device__ __forceinline__ u32x2_t int8_round8(const float (&y)[8], float s, float inv) {
  float k[8], worst = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    k[i] = rintf(y[i] * inv);
    worst = fmaxf(worst, fabsf(fmaf(-k[i], s, y[i])));
  }
  if (worst + worst >= s) {  // seldom
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float r = fmaf(-k[i], s, y[i]), twice = fabsf(r + r);
      const bool odd = fabsf(k[i] - 2.0f * rintf(0.5f * k[i])) == 1.0f;
      if (twice > s || (twice == s && odd)) k[i] += copysignf(1.0f, r);
    }
  }
  u32x2_t q;
#pragma unroll
  for (int i = 0; i < 2; ++i) {  // 1.5 2^23 + k has k's two's complement in its low bits
    constexpr float kMagic = 12582912.0f;
    const uint32_t ab = __builtin_amdgcn_perm(__float_as_uint(k[4 * i + 1] + kMagic), __float_as_uint(k[4 * i] + kMagic), 0x0c0c0400);
    const uint32_t cd = __builtin_amdgcn_perm(__float_as_uint(k[4 * i + 3] + kMagic), __float_as_uint(k[4 * i + 2] + kMagic), 0x04000c0c);
    q[i] = s == s ? ab | cd : 0;
  }
  return q;
}

// A value as it is in fp32. Without this the compiler may take a product and its conversion to fp16 as one instruction, which
// rounds once where the definition rounds twice.
__device__ __forceinline__ float as_fp32(float x) {
  asm("" : "+v"(x));
  return x;
}

}  // namespace
}  // namespace gn
