// int8.h — matrices of 8-bit integers with a scale to each row: the host entry points of int8.hip and int8_gemm.hip.
#pragma once

#include "common.h"

namespace gn {

// Sums of K products of magnitudes up to 128 x 128 stay below 2^31.
constexpr long kInt8MaxK = (1L << 17) - 1;

// Bytes from row to row of a matrix that the library lays out.
inline long int8_pitch(long cols) { return (cols + 15) / 16 * 16; }

struct Int8QuantizeDesc {
  int dtype;
  const void *x;
  long rows, cols, ldx;
  const float *col_scale;
  int8_t *q;
  long ldq;
  float *scales;
};
struct Int8GemmDesc {
  long M, N, K;
  float alpha, beta;
  const int8_t *A;
  long lda;
  const float *a_scales;
  const int8_t *B;
  long ldb;
  const float *b_scales;
  float *C;
  long ldc;
  const float *bias;
  int act;
  float act_alpha;
};
// The product with a dtype matrix of activations in A's place: gemm.A, lda and a_scales are not read.
struct Int8LinearDesc {
  int dtype;
  const void *x;
  long ldx;
  const float *col_scale;
  Int8GemmDesc gemm;
  void *workspace;
  size_t workspace_bytes;
};

// The checks need no device; the launchers expect arguments that passed them.
int check_int8_quantize(const Int8QuantizeDesc &d, CError *err);
int launch_int8_quantize(const Int8QuantizeDesc &d, hipStream_t s, CError *err);
int check_int8_dequantize(const int8_t *q, const float *scales, long rows, long cols, long ldq, int dtype,
                          const void *out, long ldo, CError *err);
int launch_int8_dequantize(const int8_t *q, const float *scales, long rows, long cols, long ldq, int dtype, void *out,
                           long ldo, hipStream_t s, CError *err);
int check_int8_gemm(const Int8GemmDesc &d, CError *err);
int launch_int8_gemm(const Int8GemmDesc &d, hipStream_t s, CError *err);
size_t int8_linear_workspace(long M, long N, long K);
int check_int8_linear(const Int8LinearDesc &d, CError *err);
int launch_int8_linear(const Int8LinearDesc &d, hipStream_t s, CError *err);

}  // namespace gn
