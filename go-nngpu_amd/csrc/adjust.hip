// adjust.hip — logits before sampling: penalties for the tokens so far, biases, masks; and the gradient of the logits.
//
// A workgroup takes a segment of a row. It counts the row's tokens that fall into the segment in LDS (whole numbers: the order
// in which they are added changes nothing), then goes once over the segment's logits, which were asked for before. Where no
// token and no bias falls into a segment the counts are not looked at.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "adjust.h"
#include "int8_round.h"

namespace gn {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxBiases = 1024;

template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

// A thread's vectors of a segment: vector i holds the segment's values at place<T>(i) and after it.
template <typename T>
__device__ __forceinline__ int place(int i) {
  return (i * kThreads + (int)threadIdx.x) * kVec<T>;
}
template <typename T>
struct Vector {
  typedef T V __attribute__((ext_vector_type(kVec<T>)));
  V v;
  // `left` values are there; those past them are 0 and are not written.
  __device__ __forceinline__ void load(const T *x, int left) {
    if (left >= kVec<T>) {
      v = __builtin_bit_cast(V, reinterpret_cast<const Unaligned16<T> *>(x)->v);
    } else {
#pragma unroll
      for (int j = 0; j < kVec<T>; ++j) v[j] = j < left ? x[j] : (T)0.0f;
    }
  }
  __device__ __forceinline__ void store(T *g, int left) const {
    if (left >= kVec<T>) {
      reinterpret_cast<Unaligned16<T> *>(g)->v = __builtin_bit_cast(u32x4_t, v);
    } else {
#pragma unroll
      for (int j = 0; j < kVec<T>; ++j)
        if (j < left) g[j] = v[j];
    }
  }
};

// The mask's bits of the kVec columns from `col` on (a multiple of kVec); all of them without a mask.
template <typename T>
__device__ __forceinline__ uint32_t allowed_bits(const uint32_t *mask, long col) {
  return mask ? mask[col >> 5] >> (col & 31) : ~0u;
}

// What a column's cell of the counts says: bit 31 in the prompt, bit 30 there is a bias, below them how often in the answer.
constexpr uint32_t kPrompt = 1u << 31, kBiased = 1u << 30, kCount = kBiased - 1;

template <typename T, int E, bool BIASES>
__global__ void __launch_bounds__(kThreads) adjust_kernel(AdjustDesc p, int segs) {
  constexpr int SEG = kThreads * E, VECS = E / kVec<T>;
  __shared__ __attribute__((aligned(16))) uint32_t cells[SEG];
  __shared__ float sums[BIASES ? SEG : 1];  // of a token's biases, where its cell says that there are some
  __shared__ int again;
  const long r = blockIdx.x / segs;
  const long col0 = (long)(blockIdx.x % segs) * SEG;
  const int left = (int)min(p.cols - col0, (long)SEG);
  const T *x = static_cast<const T *>(p.x) + r * p.ld + col0;
  T *out = static_cast<T *>(p.out) + r * p.ldo + col0;
  Vector<T> v[VECS];
#pragma unroll
  for (int i = 0; i < VECS; ++i) v[i].load(x + place<T>(i), left - place<T>(i));
#pragma unroll
  for (int i = 0; i < E / 4; ++i) reinterpret_cast<u32x4_t *>(cells)[i * kThreads + threadIdx.x] = u32x4_t{0, 0, 0, 0};
  if (threadIdx.x == 0) again = 0;
  __syncthreads();
  const long prompt = p.prompt ? p.prompt[r] : 0;
  bool any = false;
  for (long i = threadIdx.x; i < p.h; i += kThreads) {
    const uint64_t at = (uint64_t)p.history[r * p.h + i] - (uint64_t)col0;
    if (at < (uint64_t)left) {
      any = true;
      if (i < prompt)
        atomicOr(&cells[at], kPrompt);
      else
        atomicAdd(&cells[at], 1u);
    }
  }
  const int64_t *bias_ids = p.bias_ids + r * p.biases;
  const float *bias = p.bias + r * p.biases;
  if constexpr (BIASES) {
    for (int i = threadIdx.x; i < p.biases; i += kThreads) {
      const uint64_t at = (uint64_t)bias_ids[i] - (uint64_t)col0;
      if (at < (uint64_t)left) {
        any = true;
        if (atomicOr(&cells[at], kBiased) & kBiased)
          again = 1;
        else
          sums[at] = bias[i];
      }
    }
  }
  const bool touched = __syncthreads_or(any);
  // A token with several biases: its first entry's thread adds them up in order.
  if constexpr (BIASES) {
    if (again) {
      for (int i = threadIdx.x; i < p.biases; i += kThreads) {
        const uint64_t at = (uint64_t)bias_ids[i] - (uint64_t)col0;
        if (at >= (uint64_t)left) continue;
        bool first = true;
        for (int j = 0; j < i; ++j) first &= bias_ids[j] != bias_ids[i];
        if (!first) continue;
        float sum = bias[i];
        for (int j = i + 1; j < p.biases; ++j)
          if (bias_ids[j] == bias_ids[i]) sum += bias[j];
        sums[at] = sum;
      }
      __syncthreads();
    }
  }
  const float rho = p.repetition ? p.repetition[r] : 1.0f, freq = p.frequency ? p.frequency[r] : 0.0f;
  const float pres = p.presence ? p.presence[r] : 0.0f;
  const uint32_t *mask = p.mask ? p.mask + r * p.ldmask : nullptr;
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int at = place<T>(i);
    if (at >= left) break;
    const uint32_t bits = allowed_bits<T>(mask, col0 + at);
#pragma unroll
    for (int j = 0; j < kVec<T>; ++j) {
      if (touched) {
        const uint32_t cell = cells[at + j];
        if (cell != 0) {
          float y = (float)v[i].v[j];
          const uint32_t n = cell & kCount;
          if (n != 0 || (cell & kPrompt)) y = y > 0.0f ? y / rho : y * rho;
          if (n != 0) y = (y - as_fp32(freq * (float)n)) - pres;
          if (BIASES && (cell & kBiased)) y = as_fp32(y) + sums[at + j];
          v[i].v[j] = (T)as_fp32(y);
        }
      }
      if (!((bits >> j) & 1)) v[i].v[j] = (T)-INFINITY;
    }
    v[i].store(out + at, left - at);
  }
}

// The gradient of a logit is that of the adjusted one times 1, or rho or 1 / rho by the logit's sign where the token is among
// those so far, or 0 where it is masked.
template <typename T, int E>
__global__ void __launch_bounds__(kThreads) adjust_backward_kernel(AdjustGradDesc p, int segs) {
  constexpr int SEG = kThreads * E, VECS = E / kVec<T>;
  __shared__ uint32_t seen[SEG / 32];
  const long r = blockIdx.x / segs;
  const long col0 = (long)(blockIdx.x % segs) * SEG;
  const int left = (int)min(p.cols - col0, (long)SEG);
  const T *x = static_cast<const T *>(p.x) + r * p.ld + col0, *g = static_cast<const T *>(p.grad_out) + r * p.ldg + col0;
  T *out = static_cast<T *>(p.grad) + r * p.ldo + col0;
  Vector<T> v[VECS];
#pragma unroll
  for (int i = 0; i < VECS; ++i) v[i].load(g + place<T>(i), left - place<T>(i));
  bool any = false;
  if (p.repetition) {
    for (int i = threadIdx.x; i < SEG / 32; i += kThreads) seen[i] = 0;
    __syncthreads();
    for (long i = threadIdx.x; i < p.h; i += kThreads) {
      const uint64_t at = (uint64_t)p.history[r * p.h + i] - (uint64_t)col0;
      if (at < (uint64_t)left) {
        any = true;
        atomicOr(&seen[at >> 5], 1u << (at & 31));
      }
    }
  }
  const bool touched = __syncthreads_or(any);
  const float rho = p.repetition ? p.repetition[r] : 1.0f;
  const uint32_t *mask = p.mask ? p.mask + r * p.ldmask : nullptr;
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int at = place<T>(i);
    if (at >= left) break;
    const uint32_t bits = allowed_bits<T>(mask, col0 + at);
    const uint32_t hit = touched ? seen[at >> 5] >> (at & 31) : 0;
#pragma unroll
    for (int j = 0; j < kVec<T>; ++j) {
      if ((hit >> j) & 1) {
        const float d = (float)v[i].v[j];
        v[i].v[j] = (T)as_fp32((float)x[at + j] > 0.0f ? d / rho : d * rho);
      }
      if (!((bits >> j) & 1)) v[i].v[j] = (T)0.0f;
    }
    v[i].store(out + at, left - at);
  }
}

// ------------------------------------------------------------------ host
int check_rows(const char *what, const char *name, int dtype, const void *x, long rows, long cols, long ld, CError *err) {
  size_t n;
  if (ld < cols) return set_error(err, -1, "%s: leading dimension %ld of %s smaller than row length %ld", what, ld, name, cols);
  if (!matrix_bytes(rows, ld, 4, &n) || n > ((size_t)1 << 62)) return set_error(err, -1, "%s: %ld x %ld is too large", what, rows, cols);
  if (rows == 0) return 0;
  if (!x) return set_error(err, -1, "%s: NULL %s", what, name);
  if ((uintptr_t)x % (dtype == GN_F16 ? 2 : 4)) return set_error(err, -1, "%s: %s not aligned to the type", what, name);
  return 0;
}
int check_common(const char *what, int dtype, long rows, long cols, const int64_t *history, long h, const uint32_t *mask,
                 long ldmask, CError *err) {
  size_t n;
  if (dtype != GN_F32 && dtype != GN_F16) return set_error(err, -1, "%s: unsupported dtype %d", what, dtype);
  if (rows < 0 || cols < 1 || cols > INT_MAX) return set_error(err, -1, "%s: invalid size %ld x %ld", what, rows, cols);
  // A workgroup to 2048 columns and more of a row, below 2^24 of them (2^32 threads).
  if (rows >= (1L << 24) / ((cols + 8191) / 8192)) return set_error(err, -1, "%s: %ld x %ld is too large", what, rows, cols);
  // Counts stay below the bits that stand beside them.
  if (h < 0 || h >= (long)kBiased || !matrix_bytes(rows, h, 8, &n)) return set_error(err, -1, "%s: history of %ld tokens", what, h);
  if (rows == 0) return 0;
  if (h > 0 && !history) return set_error(err, -1, "%s: NULL history", what);
  if ((uintptr_t)history % 8) return set_error(err, -1, "%s: history not aligned to its type", what);
  if (mask) {
    if ((uintptr_t)mask % 4) return set_error(err, -1, "%s: mask not aligned to its type", what);
    if (ldmask < (cols + 31) / 32 || !matrix_bytes(rows, ldmask, 4, &n) || n > ((size_t)1 << 62))
      return set_error(err, -1, "%s: leading dimension %ld of the mask, %ld words are needed", what, ldmask, (cols + 31) / 32);
  }
  return 0;
}

int launched(const char *what, CError *err) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : hip_error(err, -6, what, e);
}

// Values of a row to a thread: 32, or 8 where that leaves CUs without a workgroup.
struct Split {
  int per, segs;
};
Split split_of(long rows, long cols) {
  const int per = rows * ((cols + 8191) / 8192) < 512 ? 8 : 32;
  return {per, (int)((cols + kThreads * per - 1) / (kThreads * per))};
}

// f(type, values to a thread) with both as types.
template <typename F>
void with_kind(int dtype, int per, F f) {
  using P8 = std::integral_constant<int, 8>;
  using P32 = std::integral_constant<int, 32>;
  if (dtype == GN_F16) {
    if (per == 8)
      f(_Float16{}, P8{});
    else
      f(_Float16{}, P32{});
  } else if (per == 8) {
    f(float{}, P8{});
  } else {
    f(float{}, P32{});
  }
}

}  // namespace

int check_adjust(const AdjustDesc &d, CError *err) {
  const char *what = "adjust logits";
  if (int rc = check_common(what, d.dtype, d.rows, d.cols, d.history, d.h, d.mask, d.ldmask, err)) return rc;
  if (int rc = check_rows(what, "logits", d.dtype, d.x, d.rows, d.cols, d.ld, err)) return rc;
  if (int rc = check_rows(what, "out", d.dtype, d.out, d.rows, d.cols, d.ldo, err)) return rc;
  if (d.biases < 0 || d.biases > kMaxBiases) return set_error(err, -1, "%s: 0 to %d biases to a row, got %d", what, kMaxBiases, d.biases);
  if (d.rows == 0) return 0;
  if (d.out == d.x && d.ldo != d.ld) return set_error(err, -1, "%s: in place the leading dimensions have to be equal", what);
  if (d.h == 0 && d.prompt) return set_error(err, -1, "%s: prompt lengths without a history", what);
  if ((uintptr_t)d.prompt % 8 || (uintptr_t)d.repetition % 4 || (uintptr_t)d.frequency % 4 || (uintptr_t)d.presence % 4)
    return set_error(err, -1, "%s: prompt lengths or penalties not aligned to their type", what);
  if (d.biases > 0 && (!d.bias_ids || !d.bias)) return set_error(err, -1, "%s: NULL biases", what);
  if ((uintptr_t)d.bias_ids % 8 || (uintptr_t)d.bias % 4) return set_error(err, -1, "%s: biases not aligned to their type", what);
  return 0;
}

int launch_adjust(const AdjustDesc &d, hipStream_t s, CError *err) {
  if (d.rows == 0) return 0;
  const Split sp = split_of(d.rows, d.cols);
  with_kind(d.dtype, sp.per, [&](auto type, auto per) {
    constexpr int E = decltype(per)::value;
    const dim3 grid((unsigned)(d.rows * sp.segs)), block(kThreads);
    if (d.biases > 0)
      hipLaunchKernelGGL((adjust_kernel<decltype(type), E, true>), grid, block, 0, s, d, sp.segs);
    else
      hipLaunchKernelGGL((adjust_kernel<decltype(type), E, false>), grid, block, 0, s, d, sp.segs);
  });
  return launched("adjust logits launch", err);
}

int check_adjust_backward(const AdjustGradDesc &d, CError *err) {
  const char *what = "adjust logits backward";
  if (int rc = check_common(what, d.dtype, d.rows, d.cols, d.history, d.h, d.mask, d.ldmask, err)) return rc;
  if (d.repetition && d.h > 0)  // otherwise the logits are not read
    if (int rc = check_rows(what, "logits", d.dtype, d.x, d.rows, d.cols, d.ld, err)) return rc;
  if (int rc = check_rows(what, "grad_out", d.dtype, d.grad_out, d.rows, d.cols, d.ldg, err)) return rc;
  if (int rc = check_rows(what, "grad_logits", d.dtype, d.grad, d.rows, d.cols, d.ldo, err)) return rc;
  if (d.rows == 0) return 0;
  if (d.grad == d.grad_out && d.ldo != d.ldg) return set_error(err, -1, "%s: in place the leading dimensions have to be equal", what);
  if (d.grad == d.x && d.ldo != d.ld) return set_error(err, -1, "%s: in the logits' place their leading dimension is needed", what);
  if ((uintptr_t)d.repetition % 4) return set_error(err, -1, "%s: penalties not aligned to their type", what);
  return 0;
}

int launch_adjust_backward(const AdjustGradDesc &d, hipStream_t s, CError *err) {
  if (d.rows == 0) return 0;
  const Split sp = split_of(d.rows, d.cols);
  with_kind(d.dtype, sp.per, [&](auto type, auto per) {
    hipLaunchKernelGGL((adjust_backward_kernel<decltype(type), decltype(per)::value>), dim3((unsigned)(d.rows * sp.segs)), dim3(kThreads),
                       0, s, d, sp.segs);
  });
  return launched("adjust logits backward launch", err);
}

}  // namespace gn
