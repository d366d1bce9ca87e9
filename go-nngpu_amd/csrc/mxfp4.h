// mxfp4.h — the arithmetic of MXFP4 blocks, and the host entry points of mxfp4.hip.
#pragma once

#include "common.h"

namespace gn {

constexpr int kBlock = 32;   // values to a scale
constexpr int kGroup = 128;  // values to a group of 4 blocks
__host__ __device__ inline long groups_of(long cols) { return (cols + kGroup - 1) / kGroup; }

// The scale byte of a block, from the bits of its largest magnitude (bits without the sign are ordered
// as the values are, NaN above infinity): floor(log2(top)) - 2 + 127, at least 0; 127 for a block of
// zeros, 255 for one with an infinity or NaN. The exponent field is floor(log2(top)) + 127 for a normal
// value; fp32 subnormals have field 0 and take byte 0 as all values below 2^-124 do.
__host__ __device__ inline unsigned block_scale(uint32_t top) {
  const int field = (int)(top >> 23);
  if (top == 0) return 127;
  if (field == 255) return 255;
  return (unsigned)(field > 2 ? field - 2 : 0);
}

// Whether every code times 2^(e - 127) is an fp16 value: 0.5 2^-23 (the smallest subnormal one) to 6 2^13.
constexpr unsigned kHalfLeast = 104, kHalfWidth = 36;
__host__ __device__ inline bool half_exact(unsigned e) { return e - kHalfLeast <= kHalfWidth; }

struct MxGemmDesc {
  int a_dtype;
  long M, N, K;
  float alpha, beta;
  const void *A;
  long lda;
  const void *a_scales;
  const void *B, *b_scales;
  float *C;
  long ldc;
  const float *bias;
  int act;
  float act_alpha;
};

// Bytes of a stored matrix; false for a negative size or one past 2^62 bytes.
bool mxfp4_size(long rows, long cols, size_t *data, size_t *scales);
// A stored matrix, and one of GN_F32 or GN_F16: 0, or -1 with a message.
int check_mxfp4_matrix(const char *what, const void *data, const void *scales, long rows, long cols, CError *err);
int check_plain_matrix(const char *what, int dtype, const void *x, long rows, long cols, long ld, CError *err);
// The checks need no device; the launchers expect arguments that passed them.
int check_mxfp4_quantize(int dtype, const void *x, long rows, long cols, long ldx, const void *data,
                         const void *scales, CError *err);
int launch_mxfp4_quantize(int dtype, const void *x, long rows, long cols, long ldx, void *data, void *scales,
                          hipStream_t s, CError *err);
int check_mxfp4_dequantize(const void *data, const void *scales, long rows, long cols, int dtype, const void *out,
                           long ldo, CError *err);
int launch_mxfp4_dequantize(const void *data, const void *scales, long rows, long cols, int dtype, void *out, long ldo,
                            hipStream_t s, CError *err);
int check_mxfp4_gemm(const MxGemmDesc &d, CError *err);
int launch_mxfp4_gemm(const MxGemmDesc &d, hipStream_t s, CError *err);

}  // namespace gn
