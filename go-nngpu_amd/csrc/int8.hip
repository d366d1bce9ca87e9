// int8.hip — rows of 8-bit integers with an fp32 scale each: quantisation and back (the products are in int8_gemm.hip).
//
// With y = x c (c a factor to each column, or 1) a row's scale is s = max(max |y| / 127, 2^-126) and its values the integers
// nearest to y / s, ties to even, of the exact quotient: the stored integers depend on the inputs alone, not on how a division is
// approximated.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "int8.h"
#include "int8_round.h"

namespace gn {
namespace {

constexpr long kMaxRows = (1L << 22) - 1;  // a workgroup of up to 1024 threads to a row, below 2^32 threads

struct __attribute__((packed, aligned(1))) Unaligned8 {
  u32x2_t v;
};

// ------------------------------------------------------------------ quantisation
// TX threads to a row (a wave, or a workgroup), each E times 8 values in registers, lanes next to each other on values next to
// each other: all loads in flight together, one read of the row. Longer rows (LOOP) are read twice, for their largest magnitude and
// for their values. Many rows go at the memory's rate (11008 x 4096 fp16, 135 MB, 26 to 28 us).
template <typename T, int TX, int E, bool SCALED, bool LOOP>
__global__ void __launch_bounds__(TX < 256 ? 256 : TX) int8_quantize_kernel(Int8QuantizeDesc p) {
  constexpr int RPW = TX < 256 ? 256 / TX : 1, W = TX / 64;  // rows to a workgroup, waves to a row
  __shared__ uint32_t tops[W];
  const int tx = TX < 256 ? threadIdx.x % TX : threadIdx.x;
  const long r = (long)blockIdx.x * RPW + (TX < 256 ? threadIdx.x / TX : 0);
  if (r >= p.rows) return;  // whole waves, and only where rows have no barrier
  const T *x = static_cast<const T *>(p.x) + r * p.ldx;
  // Values in their own type, or (SCALED) times their columns' factors; zeros past the row.
  using Kept = std::conditional_t<SCALED, Eight<float>, Eight<T>>;
  Kept v[E];
  auto place = [&](long c0, int e) { return c0 + 8L * (e * TX + tx); };
  auto load = [&](long c0) {
    Eight<T> raw[SCALED ? E : 1];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const long at = place(c0, e);
      if constexpr (SCALED) {
        raw[e].load(x + at, p.cols - at);
        v[e].load(p.col_scale + at, p.cols - at);
      } else {
        v[e].load(x + at, p.cols - at);
      }
    }
    if constexpr (SCALED) {
#pragma unroll
      for (int e = 0; e < E; ++e)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[e].v[i / 4][i % 4] = __float_as_uint(raw[e][i] * v[e][i]);
    }
  };
  uint32_t top = 0;
  auto reduce = [&] {
#pragma unroll
    for (int e = 0; e < E; ++e) top = max(top, v[e].top());
  };
  load(0);
  reduce();
  if constexpr (LOOP) {
    for (long c0 = 8L * TX * E; c0 < p.cols; c0 += 8L * TX * E) {
      load(c0);
      reduce();
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
  if constexpr (W > 1) {
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) top = max(top, tops[w]);
  }
  const float s = int8_scale(top), inv = 1.0f / s;
  if (tx == 0) p.scales[r] = s;
  int8_t *q = p.q + r * p.ldq;
  auto store = [&](long c0) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const long at = place(c0, e), left = p.cols - at;
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = v[e][i];
      const u32x2_t b = int8_round8(y, s, inv);
      if (left >= 8) {
        reinterpret_cast<Unaligned8 *>(q + at)->v = b;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < left) q[at + i] = (int8_t)(b[i / 4] >> (8 * (i % 4)));
      }
    }
  };
  if constexpr (LOOP) {
    for (long c0 = 0; c0 < p.cols; c0 += 8L * TX * E) {
      load(c0);
      store(c0);
    }
  } else {
    store(0);
  }
}

// ------------------------------------------------------------------ and back
// A thread takes 8 values of kRows rows, its loads in flight together; a workgroup is 1 << lx threads along a row by 256 >> lx rows.
// Memory bounds it (11008 x 4096 to fp16 21 to 22 us, half of what it reads still in the Infinity Cache after the quantisation).
constexpr int kRows = 4;

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
__global__ void __launch_bounds__(256) int8_dequantize_kernel(const int8_t *__restrict__ q, const float *__restrict__ scales,
                                                              long rows, long cols, long ldq, T *__restrict__ out, long ldo,
                                                              int lx) {
  const long at = 8L * (((long)blockIdx.y << lx) + (threadIdx.x & ((1 << lx) - 1))), left = cols - at;
  if (left <= 0) return;
  const int ry = 256 >> lx;
  const long r0 = (long)blockIdx.x * ry * kRows + (threadIdx.x >> lx);
  u32x2_t w[kRows];
  float s[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const long r = min(r0 + (long)i * ry, rows - 1);
    const int8_t *b = q + r * ldq + at;
    if (left >= 8) {
      w[i] = reinterpret_cast<const Unaligned8 *>(b)->v;
    } else {
      w[i] = u32x2_t{0, 0};
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < left) w[i][j / 4] |= (uint32_t)(uint8_t)b[j] << (8 * (j % 4));
    }
    s[i] = scales[r];
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const long r = r0 + (long)i * ry;
    if (r >= rows) break;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = as_fp32((float)(int8_t)(w[i][j / 4] >> (8 * (j % 4))) * s[i]);
    store8(out + r * ldo + at, left, v);
  }
}

int launched(const char *what, CError *err) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : hip_error(err, -6, what, e);
}

int check_plain(const char *what, int dtype, const void *x, long rows, long cols, long ld, CError *err) {
  size_t n;
  if (dtype != GN_F32 && dtype != GN_F16) return set_error(err, -1, "%s: unsupported dtype %d", what, dtype);
  if (rows < 0 || cols < 0 || !matrix_bytes(rows, ld < 0 ? 0 : ld, 4, &n) || n > ((size_t)1 << 62))
    return set_error(err, -1, "%s: invalid size %ld x %ld", what, rows, cols);
  // 65535 grid rows of 2048 columns.
  if (rows > kMaxRows || cols > 65535L * 2048) return set_error(err, -1, "%s: %ld x %ld is too large", what, rows, cols);
  if (rows == 0) return 0;
  if (ld < cols) return set_error(err, -1, "%s: leading dimension %ld smaller than row length %ld", what, ld, cols);
  if (cols == 0) return 0;
  if (!x) return set_error(err, -1, "%s: NULL matrix", what);
  if ((uintptr_t)x % (dtype == GN_F16 ? 2 : 4)) return set_error(err, -1, "%s: matrix not aligned to its type", what);
  return 0;
}
int check_stored(const char *what, const void *q, const float *scales, long rows, long cols, long ldq, CError *err) {
  size_t n;
  if (rows == 0) return 0;
  if (ldq < cols || !matrix_bytes(rows, ldq, 1, &n) || n > ((size_t)1 << 62))
    return set_error(err, -1, "%s: leading dimension %ld of the int8 matrix for %ld x %ld", what, ldq, rows, cols);
  if ((!q && cols > 0) || !scales) return set_error(err, -1, "%s: NULL int8 matrix or scales", what);
  if ((uintptr_t)scales % 4) return set_error(err, -1, "%s: scales not aligned to fp32", what);
  return 0;
}

template <typename T, bool SCALED>
void launch_rows(const Int8QuantizeDesc &d, hipStream_t s) {
  auto go = [&](auto tx, auto e, auto loop) {
    constexpr int TX = decltype(tx)::value, E = decltype(e)::value, NT = TX < 256 ? 256 : TX;
    hipLaunchKernelGGL((int8_quantize_kernel<T, TX, E, SCALED, decltype(loop)::value>),
                       dim3((unsigned)((d.rows * TX + NT - 1) / NT)), dim3(NT), 0, s, d);
  };
  using std::integral_constant;
  // As few threads as take the row at once with little left over. Measured, us: 4096 rows of 1000 fp32 a wave 5.6, 256 threads 7.1; 512 of 4096
  // fp16 256 x 16 values 3.7, 256 x 32 4.7, 1024 x 8 4.3; 11008 of 4096 23, 29 and 48 (5.9 TB/s); 8192 of 8192 256 x 32 37, 512 x 16 37, 1024 x 8
  // 44; 512 of 11008 fp32 with factors 512 x 32 7.7, 1024 x 16 7.7, 1024 x 32 12.
  if (d.cols <= 512)
    go(integral_constant<int, 64>{}, integral_constant<int, 1>{}, std::false_type{});
  else if (d.cols <= 1024)
    go(integral_constant<int, 64>{}, integral_constant<int, 2>{}, std::false_type{});
  else if (d.cols <= 2048)
    go(integral_constant<int, 256>{}, integral_constant<int, 1>{}, std::false_type{});
  else if (d.cols <= 4096)
    go(integral_constant<int, 256>{}, integral_constant<int, 2>{}, std::false_type{});
  else if (d.cols <= 8192)
    go(integral_constant<int, 512>{}, integral_constant<int, 2>{}, std::false_type{});
  else if (d.cols <= 16384)
    go(integral_constant<int, 512>{}, integral_constant<int, 4>{}, std::false_type{});
  else if (d.cols <= 32768)
    go(integral_constant<int, 1024>{}, integral_constant<int, 4>{}, std::false_type{});
  else
    go(integral_constant<int, 1024>{}, integral_constant<int, 4>{}, std::true_type{});
}

}  // namespace

int check_int8_quantize(const Int8QuantizeDesc &d, CError *err) {
  const char *what = "int8 quantize";
  if (int rc = check_plain(what, d.dtype, d.x, d.rows, d.cols, d.ldx, err)) return rc;
  if ((uintptr_t)d.col_scale % 4) return set_error(err, -1, "%s: column factors not aligned to fp32", what);
  return check_stored(what, d.q, d.scales, d.rows, d.cols, d.ldq, err);
}

int launch_int8_quantize(const Int8QuantizeDesc &d, hipStream_t s, CError *err) {
  if (d.rows == 0) return 0;
  if (d.dtype == GN_F16)
    d.col_scale ? launch_rows<_Float16, true>(d, s) : launch_rows<_Float16, false>(d, s);
  else
    d.col_scale ? launch_rows<float, true>(d, s) : launch_rows<float, false>(d, s);
  return launched("int8 quantize launch", err);
}

int check_int8_dequantize(const int8_t *q, const float *scales, long rows, long cols, long ldq, int dtype,
                          const void *out, long ldo, CError *err) {
  const char *what = "int8 dequantize";
  if (int rc = check_plain(what, dtype, out, rows, cols, ldo, err)) return rc;
  return cols == 0 ? 0 : check_stored(what, q, scales, rows, cols, ldq, err);
}

int launch_int8_dequantize(const int8_t *q, const float *scales, long rows, long cols, long ldq, int dtype, void *out,
                           long ldo, hipStream_t s, CError *err) {
  if (rows == 0 || cols == 0) return 0;
  const long words = (cols + 7) / 8;
  int lx = 4;
  while (lx < 8 && (1 << lx) < words) ++lx;
  const long per = (256 >> lx) * kRows;
  const dim3 grid((unsigned)((rows + per - 1) / per), (unsigned)((words + (1 << lx) - 1) >> lx));
  if (dtype == GN_F16)
    hipLaunchKernelGGL(int8_dequantize_kernel<_Float16>, grid, dim3(256), 0, s, q, scales, rows, cols, ldq,
                       static_cast<_Float16 *>(out), ldo, lx);
  else
    hipLaunchKernelGGL(int8_dequantize_kernel<float>, grid, dim3(256), 0, s, q, scales, rows, cols, ldq,
                       static_cast<float *>(out), ldo, lx);
  return launched("int8 dequantize launch", err);
}

}  // namespace gn
