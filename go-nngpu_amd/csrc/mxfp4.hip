// mxfp4.hip — MXFP4 matrices: quantisation, dequantisation and the product with 4-bit weights.
//
// A block of 32 values along a row has one scale byte E (2^(E - 127), 255 for NaN) and 32 e2m1
// codes in 16 bytes. Rows are stored in whole groups of 128 values (64 bytes of codes, one dword of
// scales): the K of one v_mfma_scale_f32_16x16x128, whose lane l takes the block l / 16 of row
// l % 16, so both operands are read in their stored order.
#include "gemm_tile.h"
#include "mxfp4.h"

namespace gn {
namespace {

constexpr int kBlock = 32;   // values to a scale
constexpr int kGroup = 128;  // values to a group of 4 blocks

typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef float float2_t __attribute__((ext_vector_type(2)));

__host__ __device__ inline long groups_of(long cols) { return (cols + kGroup - 1) / kGroup; }

// 2^(E - 127); NaN for 255.
__device__ __forceinline__ float scale_of(unsigned e) {
  return __uint_as_float((e << 23) | ((e == 0 || e == 255) ? 0x00400000u : 0u));
}

// ------------------------------------------------------------------ quantisation
// A thread owns a word of codes: 8 values, a quarter of a block, so that lanes next to each other read
// and write next to each other. A workgroup is TX = 1 << lx threads along a row (the power of two at or
// above the row's words, at most 256) by 256 >> lx rows, and takes kRows such sets of rows with their
// loads in flight together; 32-bit shifts stand in for the division of an index by the row length.
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

// ------------------------------------------------------------------ product
struct MxParams {
  const void *A;
  const uint8_t *as;
  const u32x4_t *B;
  const uint8_t *bs;
  float *C;
  const float *bias;
  long M, N, K, lda, ldc;
  float alpha, beta, act_alpha;
  int act;
};

__device__ __forceinline__ float4_t mfma_fp4(u32x4_t a, u32x4_t b, float4_t c, int sa, int sb) {
  const i32x8_t x = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  const i32x8_t y = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 4, 4, 0, sa, 0, sb);
}

// Eight codes as halves, times 2^(exponent of unit - 127).
__device__ __forceinline__ half8_t half8_of(uint32_t w, float unit) {
  const half2_t a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, unit, 0);
  const half2_t b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, unit, 1);
  const half2_t c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, unit, 2);
  const half2_t d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, unit, 3);
  return half8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

__device__ __forceinline__ float finish(const MxParams &p, float acc, long m, long n) {
  float v = p.alpha * acc;
  if (p.beta != 0.0f) v += p.beta * p.C[m * p.ldc + n];
  if (p.bias) v += p.bias[n];
  return apply_act(p.act, v, p.act_alpha);
}

// One wave per 16 x 16 tile, operands from global memory.
template <bool FP4>
__global__ void __launch_bounds__(64) mx_tile_kernel(MxParams p) {
  const int lane = threadIdx.x, l16 = lane & 15, g = lane >> 4;
  const long tn = (p.N + 15) / 16, m0 = blockIdx.x / tn * 16, n0 = blockIdx.x % tn * 16;
  const long am = min(m0 + l16, p.M - 1), bn = min(n0 + l16, p.N - 1), G = groups_of(p.K);
  const u32x4_t *b = p.B + bn * G * 4 + g;
  const uint32_t *bs = reinterpret_cast<const uint32_t *>(p.bs) + bn * G;
  float4_t acc = {0, 0, 0, 0};
  for (long c = 0; c < G; ++c) {
    const u32x4_t bq = b[c * 4];
    const uint32_t bsc = bs[c];
    if constexpr (FP4) {
      const u32x4_t aq = (static_cast<const u32x4_t *>(p.A) + am * G * 4 + g)[c * 4];
      const uint32_t asc = (reinterpret_cast<const uint32_t *>(p.as) + am * G)[c];
      acc = mfma_fp4(aq, bq, acc, asc >> (8 * g), bsc >> (8 * g));
    } else {
      const _Float16 *a = static_cast<const _Float16 *>(p.A) + am * p.lda;
      half8_t av[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const long k = c * kGroup + g * kBlock + j * 8 + e;
          av[j][e] = k < p.K ? a[k] : (_Float16)0;
        }
      const unsigned e = (bsc >> (8 * g)) & 255;
      if (__all(half_exact(e))) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(av[j], half8_of(bq[j], scale_of(e)), acc, 0, 0, 0);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) {  // block q of both sides, the rest zeros
          float4_t part = {0, 0, 0, 0};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const half8_t z = {0, 0, 0, 0, 0, 0, 0, 0};
            part = __builtin_amdgcn_mfma_f32_16x16x32_f16(g == q ? av[j] : z, g == q ? half8_of(bq[j], 1.0f) : z, part,
                                                          0, 0, 0);
          }
          const float unit = scale_of((bsc >> (8 * q)) & 255);
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[i] = fmaf(part[i], unit, acc[i]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long m = m0 + 4 * g + i, n = n0 + l16;
    if (m < p.M && n < p.N) p.C[m * p.ldc + n] = finish(p, acc[i], m, n);
  }
}

// K == 0: act(beta C + bias).
__global__ void __launch_bounds__(256) mx_k0_kernel(MxParams p) {
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < p.M * p.N; i += (long)gridDim.x * 256)
    p.C[i / p.N * p.ldc + i % p.N] = finish(p, 0.0f, i / p.N, i % p.N);
}

int check_matrix(const char *what, const void *data, const void *scales, long rows, long cols, CError *err) {
  size_t d, s;
  if (!mxfp4_size(rows, cols, &d, &s)) return set_error(err, -1, "%s: invalid size %ld x %ld", what, rows, cols);
  if (d == 0) return 0;
  if (!data || !scales) return set_error(err, -1, "%s: NULL data or scales", what);
  if ((uintptr_t)data % 16 || (uintptr_t)scales % 4)
    return set_error(err, -1, "%s: data at a multiple of 16 bytes and scales at one of 4 are needed", what);
  return 0;
}

int check_plain(const char *what, int dtype, const void *x, long rows, long cols, long ld, CError *err) {
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

unsigned grid_of(long n, long per) { return (unsigned)std::max(1L, std::min((n + per - 1) / per, 1L << 20)); }

}  // namespace

bool mxfp4_size(long rows, long cols, size_t *data, size_t *scales) {
  if (rows < 0 || cols < 0 || cols > LONG_MAX - kGroup) return false;
  size_t n;
  if (!matrix_bytes(rows, groups_of(cols), 256, &n) || n > ((size_t)1 << 62)) return false;  // offsets stay in 63 bits
  *data = n / 4;
  *scales = n / 64;
  return true;
}

int check_mxfp4_quantize(int dtype, const void *x, long rows, long cols, long ldx, const void *data,
                         const void *scales, CError *err) {
  if (int rc = check_plain("mxfp4 quantize", dtype, x, rows, cols, ldx, err)) return rc;
  if (cols > kMaxCols || rows > kMaxRows) return set_error(err, -1, "mxfp4 quantize: %ld x %ld is too large", rows, cols);
  return check_matrix("mxfp4 quantize", data, scales, rows, cols, err);
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
  if (int rc = check_plain("mxfp4 dequantize", dtype, out, rows, cols, ldo, err)) return rc;
  if (cols > kMaxCols || rows > kMaxRows) return set_error(err, -1, "mxfp4 dequantize: %ld x %ld is too large", rows, cols);
  return check_matrix("mxfp4 dequantize", data, scales, rows, cols, err);
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

int check_mxfp4_gemm(const MxGemmDesc &d, CError *err) {
  if (d.a_dtype != GN_F16 && d.a_dtype != GN_MXFP4)
    return set_error(err, -1, "mxfp4 gemm: unsupported dtype %d of A", d.a_dtype);
  size_t n;
  if (d.M < 0 || d.N < 0 || d.K < 0) return set_error(err, -1, "mxfp4 gemm: negative size");
  if (!act_supported(d.act)) return set_error(err, -1, "mxfp4 gemm: unsupported activation %d", d.act);
  if (d.M == 0 || d.N == 0) return 0;
  if (!d.C) return set_error(err, -1, "mxfp4 gemm: NULL C");
  if (d.ldc < d.N) return set_error(err, -1, "mxfp4 gemm: leading dimension smaller than row length");
  if ((uintptr_t)d.C % 4 || (uintptr_t)d.bias % 4) return set_error(err, -1, "mxfp4 gemm: C or bias not aligned to fp32");
  if (!matrix_bytes(d.M, d.ldc, 4, &n) || n > ((size_t)1 << 62) || (d.M + 15) / 16 > (1L << 26) / ((d.N + 15) / 16))
    return set_error(err, -1, "mxfp4 gemm: problem too large for the grid");
  if (d.K == 0) return 0;
  if (int rc = check_matrix("mxfp4 gemm: B", d.B, d.b_scales, d.N, d.K, err)) return rc;
  if (d.a_dtype == GN_MXFP4) return check_matrix("mxfp4 gemm: A", d.A, d.a_scales, d.M, d.K, err);
  if (d.a_scales) return set_error(err, -1, "mxfp4 gemm: scales given for an fp16 A");
  return check_plain("mxfp4 gemm: A", GN_F16, d.A, d.M, d.K, d.lda, err);
}

int launch_mxfp4_gemm(const MxGemmDesc &d, hipStream_t s, CError *err) {
  if (d.M == 0 || d.N == 0) return 0;
  MxParams p{};
  p.A = d.A;
  p.as = static_cast<const uint8_t *>(d.a_scales);
  p.B = static_cast<const u32x4_t *>(d.B);
  p.bs = static_cast<const uint8_t *>(d.b_scales);
  p.C = d.C;
  p.bias = d.bias;
  p.M = d.M, p.N = d.N, p.K = d.K, p.lda = d.lda, p.ldc = d.ldc;
  p.alpha = d.alpha, p.beta = d.beta, p.act = d.act, p.act_alpha = d.act_alpha;
  if (d.K == 0) {
    hipLaunchKernelGGL(mx_k0_kernel, dim3(grid_of(d.M * d.N, 256)), dim3(256), 0, s, p);
  } else {
    const dim3 grid((unsigned)(((d.M + 15) / 16) * ((d.N + 15) / 16)));
    if (d.a_dtype == GN_MXFP4)
      hipLaunchKernelGGL(mx_tile_kernel<true>, grid, dim3(64), 0, s, p);
    else
      hipLaunchKernelGGL(mx_tile_kernel<false>, grid, dim3(64), 0, s, p);
  }
  return launched("mxfp4 gemm launch", err);
}

}  // namespace gn
