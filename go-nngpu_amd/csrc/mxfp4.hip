// mxfp4.hip — MXFP4 matrices: their storage, quantisation and dequantisation (the products are in mxfp4_gemm.hip).
//
// A block of 32 values along a row has one scale byte E (2^(E - 127), 255 for NaN) and 32 e2m1
// codes in 16 bytes. Rows are stored in whole groups of 128 values (64 bytes of codes, one dword of
// scales).
#include <algorithm>
#include <climits>

#include "mxfp4.h"

namespace gn {
namespace {

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------ quantisation
// A thread owns a word of codes: 8 values, a quarter of a block, so that lanes next to each other read
// and write next to each other. A workgroup is TX = 1 << lx threads along a row (the power of two at or
// above the row's words, at most 256) by 256 >> lx rows, and takes kRows such sets of rows with their
// loads in flight together; 32-bit shifts stand in for the division of an index by the row length.
// Bound by memory: 8192 x 8192 fp16 to 4 bits takes 29 us (5.8 TB/s read and written; a large copy reaches 4.6, its lines not
// kept in the last-level cache).
constexpr int kRows = 4;
// 65535 grid rows of 2048 columns, and grid columns of at least 4 rows and 256 threads, below 2^32 threads in all.
constexpr long kMaxCols = 65535L * 2048, kMaxRows = 1L << 25;

// 16 bytes at any address that is a multiple of T's size (the hardware takes unaligned vectors).
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Unaligned16 {
  u32x4_t v;
};

// Eight values from p as fp32, 0 for those at or past `left`.
__device__ __forceinline__ void load8(const float *p, long left, float v[8]) {
  if (left >= 8) {
    const u32x4_t a = reinterpret_cast<const Unaligned16<float> *>(p)[0].v;
    const u32x4_t b = reinterpret_cast<const Unaligned16<float> *>(p)[1].v;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(a[j]), v[j + 4] = __uint_as_float(b[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < left ? p[j] : 0.0f;
  }
}
__device__ __forceinline__ void load8(const _Float16 *p, long left, float v[8]) {
  if (left >= 8) {
    const u32x4_t a = reinterpret_cast<const Unaligned16<_Float16> *>(p)->v;
    const half8_t h = __builtin_bit_cast(half8_t, a);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (float)h[j];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < left ? (float)p[j] : 0.0f;
  }
}

template <typename T>
__global__ void __launch_bounds__(256) quantize_kernel(const T *__restrict__ x, long rows, long cols, long ldx,
                                                       uint32_t *__restrict__ data, uint8_t *__restrict__ scales,
                                                       int words, int lx) {
  const int w = (blockIdx.y << lx) + (threadIdx.x & ((1 << lx) - 1));
  if (w >= words) return;  // words is a multiple of 16: the four lanes of a block leave together
  const int ry = 256 >> lx;
  const long r0 = (long)blockIdx.x * ry * kRows + (threadIdx.x >> lx), left = cols - 8L * w;
  float v[kRows][8];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const long r = min(r0 + (long)i * ry, rows - 1);
    load8(x + r * ldx + 8L * w, left, v[i]);
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const long r = r0 + (long)i * ry;
    uint32_t top = 0;  // the bits of non-negative floats are ordered as their values, NaN above infinity
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[i][j]) & 0x7fffffffu);
    top = max(top, (uint32_t)__shfl_xor((int)top, 1, 64));
    top = max(top, (uint32_t)__shfl_xor((int)top, 2, 64));
    const unsigned e = block_scale(top);
    // The conversion divides by 2^(e - 127), taken from its operand's exponent field (0 included), rounds
    // to nearest even and saturates.
    const float unit = __uint_as_float(e << 23);
    uint32_t q = 0;
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[i][0], v[i][1], unit, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[i][2], v[i][3], unit, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[i][4], v[i][5], unit, 2);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[i][6], v[i][7], unit, 3);
    if (r < rows) {
      data[r * words + w] = e == 255 ? 0u : q;
      if ((w & 3) == 0) scales[(r * words + w) >> 2] = (uint8_t)e;
    }
  }
}

__device__ __forceinline__ void store8(float *p, long left, const float v[8]) {
  if (left >= 8) {
    u32x4_t a, b;
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = __float_as_uint(v[j]), b[j] = __float_as_uint(v[j + 4]);
    reinterpret_cast<Unaligned16<float> *>(p)[0].v = a;
    reinterpret_cast<Unaligned16<float> *>(p)[1].v = b;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < left) p[j] = v[j];
  }
}
__device__ __forceinline__ void store8(_Float16 *p, long left, const float v[8]) {
  half8_t h;
#pragma unroll
  for (int j = 0; j < 8; ++j) h[j] = (_Float16)v[j];
  if (left >= 8) {
    reinterpret_cast<Unaligned16<_Float16> *>(p)->v = __builtin_bit_cast(u32x4_t, h);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < left) p[j] = h[j];
  }
}

template <typename T>
__global__ void __launch_bounds__(256) dequantize_kernel(const uint32_t *__restrict__ data,
                                                         const uint8_t *__restrict__ scales, long rows, long cols,
                                                         T *__restrict__ out, long ldo, int words, int lx) {
  const int w = (blockIdx.y << lx) + (threadIdx.x & ((1 << lx) - 1));
  const long left = cols - 8L * w;
  if (left <= 0) return;
  const int ry = 256 >> lx;
  const long r0 = (long)blockIdx.x * ry * kRows + (threadIdx.x >> lx);
  uint32_t q[kRows];
  unsigned e[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const long r = min(r0 + (long)i * ry, rows - 1);
    q[i] = data[r * words + w];
    e[i] = scales[(r * words + w) >> 2];
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const long r = r0 + (long)i * ry;
    if (r >= rows) break;
    const float unit = __uint_as_float(e[i] << 23);
    float v[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float2_t f;
      if (j == 0) f = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[i], unit, 0);
      if (j == 1) f = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[i], unit, 1);
      if (j == 2) f = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[i], unit, 2);
      if (j == 3) f = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[i], unit, 3);
      v[2 * j] = e[i] == 255 ? NAN : f[0];
      v[2 * j + 1] = e[i] == 255 ? NAN : f[1];
    }
    store8(out + r * ldo + 8L * w, left, v);
  }
}

int launched(const char *what, CError *err) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : hip_error(err, -6, what, e);
}

struct WordGrid {
  dim3 grid;
  int words, lx;
};
WordGrid word_grid(long rows, long cols) {
  WordGrid w;
  w.words = (int)(groups_of(cols) * 16);
  for (w.lx = 4; w.lx < 8 && (1 << w.lx) < w.words; ++w.lx) {}
  const long per = (256 >> w.lx) * kRows;
  w.grid = dim3((unsigned)((rows + per - 1) / per), (unsigned)((w.words + (1 << w.lx) - 1) >> w.lx));
  return w;
}

}  // namespace

bool mxfp4_size(long rows, long cols, size_t *data, size_t *scales) {
  if (rows < 0 || cols < 0 || cols > LONG_MAX - kGroup) return false;
  size_t n;
  if (!matrix_bytes(rows, groups_of(cols), 256, &n) || n > ((size_t)1 << 62)) return false;  // offsets stay in 63 bits
  *data = n / 4;
  *scales = n / 64;
  return true;
}

int check_mxfp4_matrix(const char *what, const void *data, const void *scales, long rows, long cols, CError *err) {
  size_t d, s;
  if (!mxfp4_size(rows, cols, &d, &s)) return set_error(err, -1, "%s: invalid size %ld x %ld", what, rows, cols);
  if (d == 0) return 0;
  if (!data || !scales) return set_error(err, -1, "%s: NULL data or scales", what);
  if ((uintptr_t)data % 16 || (uintptr_t)scales % 4)
    return set_error(err, -1, "%s: data at a multiple of 16 bytes and scales at one of 4 are needed", what);
  return 0;
}

int check_plain_matrix(const char *what, int dtype, const void *x, long rows, long cols, long ld, CError *err) {
  size_t n;
  if (dtype != GN_F32 && dtype != GN_F16) return set_error(err, -1, "%s: unsupported dtype %d", what, dtype);
  if (rows < 0 || cols < 0 || !matrix_bytes(rows, ld < 0 ? 0 : ld, 4, &n) || n > ((size_t)1 << 62))
    return set_error(err, -1, "%s: invalid size %ld x %ld", what, rows, cols);
  if (rows == 0 || cols == 0) return 0;
  if (ld < cols) return set_error(err, -1, "%s: leading dimension %ld smaller than row length %ld", what, ld, cols);
  if (!x) return set_error(err, -1, "%s: NULL matrix", what);
  if ((uintptr_t)x % (dtype == GN_F16 ? 2 : 4)) return set_error(err, -1, "%s: matrix not aligned to its type", what);
  return 0;
}

int check_mxfp4_quantize(int dtype, const void *x, long rows, long cols, long ldx, const void *data,
                         const void *scales, CError *err) {
  if (int rc = check_plain_matrix("mxfp4 quantize", dtype, x, rows, cols, ldx, err)) return rc;
  if (cols > kMaxCols || rows > kMaxRows) return set_error(err, -1, "mxfp4 quantize: %ld x %ld is too large", rows, cols);
  return check_mxfp4_matrix("mxfp4 quantize", data, scales, rows, cols, err);
}

int launch_mxfp4_quantize(int dtype, const void *x, long rows, long cols, long ldx, void *data, void *scales,
                          hipStream_t s, CError *err) {
  if (rows == 0 || cols == 0) return 0;
  const WordGrid w = word_grid(rows, cols);
  auto *d = static_cast<uint32_t *>(data);
  auto *sc = static_cast<uint8_t *>(scales);
  if (dtype == GN_F16)
    hipLaunchKernelGGL(quantize_kernel<_Float16>, w.grid, dim3(256), 0, s, static_cast<const _Float16 *>(x), rows,
                       cols, ldx, d, sc, w.words, w.lx);
  else
    hipLaunchKernelGGL(quantize_kernel<float>, w.grid, dim3(256), 0, s, static_cast<const float *>(x), rows, cols,
                       ldx, d, sc, w.words, w.lx);
  return launched("mxfp4 quantize launch", err);
}

int check_mxfp4_dequantize(const void *data, const void *scales, long rows, long cols, int dtype, const void *out,
                           long ldo, CError *err) {
  if (int rc = check_plain_matrix("mxfp4 dequantize", dtype, out, rows, cols, ldo, err)) return rc;
  if (cols > kMaxCols || rows > kMaxRows) return set_error(err, -1, "mxfp4 dequantize: %ld x %ld is too large", rows, cols);
  return check_mxfp4_matrix("mxfp4 dequantize", data, scales, rows, cols, err);
}

int launch_mxfp4_dequantize(const void *data, const void *scales, long rows, long cols, int dtype, void *out, long ldo,
                            hipStream_t s, CError *err) {
  if (rows == 0 || cols == 0) return 0;
  const WordGrid w = word_grid(rows, cols);
  auto *d = static_cast<const uint32_t *>(data);
  auto *sc = static_cast<const uint8_t *>(scales);
  if (dtype == GN_F16)
    hipLaunchKernelGGL(dequantize_kernel<_Float16>, w.grid, dim3(256), 0, s, d, sc, rows, cols,
                       static_cast<_Float16 *>(out), ldo, w.words, w.lx);
  else
    hipLaunchKernelGGL(dequantize_kernel<float>, w.grid, dim3(256), 0, s, d, sc, rows, cols,
                       static_cast<float *>(out), ldo, w.words, w.lx);
  return launched("mxfp4 dequantize launch", err);
}

}  // namespace gn
