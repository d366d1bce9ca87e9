// logits.hip — rows of logits: log-sum-exp, log-probabilities of given tokens, entropy, the top
// alternatives, distillation from a teacher's top logits, and the gradients of the logits.
//
// With z = x / T, m = max z, s = sum e^(z - m) and t = sum (z - m) e^(z - m): lse = m + ln s and the entropy is
// ln s - t / s, two terms that are never negative (no cancellation). All sums are fp32.
#include <climits>

#include "logits.h"

namespace gn {
namespace {

constexpr int kThreads = 256;
constexpr float kLog2e = 1.44269504088896340736f;

// Order of the top alternatives: the larger value first, then the lower column. A float's bits as an
// unsigned number that is ordered as the values are (NaN above infinity, -0 as 0).
__device__ __forceinline__ uint32_t value_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  if ((b & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  if (k == 0xffffffffu) return NAN;
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ uint64_t entry_key(float x, uint32_t col) { return ((uint64_t)value_key(x) << 32) | ~col; }

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int o) {
  return ((uint64_t)(uint32_t)__shfl_xor((int)(v >> 32), o, 64) << 32) | (uint32_t)__shfl_xor((int)v, o, 64);
}

// Over the workgroup's threads; every thread gets the result. red: one value for each wave.
template <typename T, typename F>
__device__ __forceinline__ T block_all(T v, T *red, F op) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    if constexpr (sizeof(T) == 8)
      v = op(v, (T)shfl_xor64((uint64_t)v, o));
    else
      v = op(v, __shfl_xor(v, o, 64));
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
  for (int i = 1; i < kThreads / 64; ++i) v = op(v, red[i]);
  return v;
}

struct RowStats {
  float m, s, t;  // max z; sums of e^(z - m) and (z - m) e^(z - m)
};

// One workgroup per row.
template <typename T>
__device__ __forceinline__ RowStats row_stats(const T *x, long cols, float inv_t, float *red) {
  auto fmax2 = [](float a, float b) { return fmaxf(a, b); };
  auto add2 = [](float a, float b) { return a + b; };
  RowStats r{-INFINITY, 0.0f, 0.0f};
  for (long i = threadIdx.x; i < cols; i += kThreads) r.m = fmaxf(r.m, (float)x[i] * inv_t);
  r.m = block_all(r.m, red, fmax2);
  const float m = r.m == -INFINITY ? 0.0f : r.m;  // a row of -inf: all terms e^-inf = 0
  for (long i = threadIdx.x; i < cols; i += kThreads) {
    const float d = (float)x[i] * inv_t - m, e = expf(d);
    r.s += e;
    if (e != 0.0f) r.t += e * d;  // also where e is NaN
  }
  r.s = block_all(r.s, red, add2);
  r.t = block_all(r.t, red, add2);
  return r;
}
__device__ __forceinline__ float lse_of(const RowStats &r) { return r.s == 0.0f ? -INFINITY : r.m + logf(r.s); }
__device__ __forceinline__ float entropy_of(const RowStats &r) { return r.s == 0.0f ? 0.0f : logf(r.s) - r.t / r.s; }
__device__ __forceinline__ float logprob_of(float z, float lse) { return lse == -INFINITY ? -INFINITY : z - lse; }

template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_kernel(LogprobsDesc p, float inv_t) {
  __shared__ float red[kThreads / 64];
  __shared__ uint64_t red64[kThreads / 64];
  for (long r = blockIdx.x; r < p.in.rows; r += gridDim.x) {
    const T *x = static_cast<const T *>(p.in.x) + r * p.in.ld;
    const RowStats st = row_stats(x, p.in.cols, inv_t, red);
    const float lse = lse_of(st);
    if (threadIdx.x == 0) {
      if (p.lse) p.lse[r] = lse;
      if (p.entropy) p.entropy[r] = entropy_of(st);
      if (p.targets) {
        const long t = p.targets[r];
        p.logprob[r] = t < 0 ? 0.0f : t >= p.in.cols ? NAN : logprob_of((float)x[t] * inv_t, lse);
      }
    }
    uint64_t last = ~0ull;
    for (int i = 0; i < p.k; ++i) {
      uint64_t best = 0;
      for (long c = threadIdx.x; c < p.in.cols; c += kThreads) {
        const uint64_t key = entry_key((float)x[c], (uint32_t)c);
        if (key < last && key > best) best = key;
      }
      last = block_all(best, red64, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
      if (threadIdx.x == 0) {
        p.top_ids[r * p.k + i] = (int64_t)(uint32_t)~last;
        p.top_logprobs[r * p.k + i] = logprob_of(key_value((uint32_t)(last >> 32)) * inv_t, lse);
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_backward_kernel(LogprobsGradDesc p, float inv_t) {
  for (long r = blockIdx.x; r < p.in.rows; r += gridDim.x) {
    const T *x = static_cast<const T *>(p.in.x) + r * p.in.ld;
    T *g = static_cast<T *>(p.grad) + r * p.ldg;
    const long t = p.targets ? p.targets[r] : -1;
    float gl = t >= 0 ? p.grad_logprob[r] : 0.0f;
    if (t >= p.in.cols) gl = NAN;
    const float gh = p.grad_entropy ? p.grad_entropy[r] : 0.0f, h = p.grad_entropy ? p.entropy[r] : 0.0f;
    const float lse = p.lse[r];
    const bool none = (gl == 0.0f && gh == 0.0f) || (lse == -INFINITY && t < p.in.cols);
    for (long c = threadIdx.x; c < p.in.cols; c += kThreads) {
      float v = 0.0f;
      if (!none) {
        const float lp = (float)x[c] * inv_t - lse, q = expf(lp);
        v = -q * gl;
        if (q != 0.0f) v -= gh * q * (lp + h);
        if (c == t) v += gl;
        v *= inv_t;
      }
      g[c] = (T)v;
    }
  }
}

// The teacher's distribution over its k entries, in w (and the ids in at): w = 0 for absent ones. Returns
// false for a row without entries; w is NaN throughout where an id is too large or a logit is NaN or +inf.
__device__ __forceinline__ bool teacher_row(const DistillDesc &p, long r, float inv_t, float *w, float *lw, int64_t *at,
                                            float *red) {
  const int i = threadIdx.x;
  int64_t id = -1;
  float z = -INFINITY;
  if (i < p.k) {
    id = p.ids[r * p.k + i];
    const float t = p.teacher[r * p.k + i];
    if (id >= p.in.cols)
      z = NAN, id = -1;
    else if (id >= 0)
      z = t * inv_t;
    if (z == -INFINITY) id = -1;
  }
  const float m = block_all(z, red, [](float a, float b) { return a != a || b != b ? NAN : fmaxf(a, b); });
  if (m == -INFINITY) return false;
  const float e = z == -INFINITY ? 0.0f : expf(z - m);
  const float s = block_all(e, red, [](float a, float b) { return a + b; });
  if (i < p.k) {
    w[i] = e / s;
    lw[i] = z - m - logf(s);
    at[i] = id;
  }
  __syncthreads();
  return true;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) distill_kernel(DistillDesc p, float inv_t) {
  __shared__ float red[kThreads / 64], w[kTeacherMax], lw[kTeacherMax];
  __shared__ int64_t at[kTeacherMax];
  for (long r = blockIdx.x; r < p.in.rows; r += gridDim.x) {
    const T *x = static_cast<const T *>(p.in.x) + r * p.in.ld;
    const RowStats st = row_stats(x, p.in.cols, inv_t, red);
    const float lse = lse_of(st);
    const bool some = teacher_row(p, r, inv_t, w, lw, at, red);
    float part = 0.0f;
    const int i = threadIdx.x;
    if (some && i < p.k) {
      if (w[i] != w[i])
        part = NAN;
      else if (at[i] >= 0 && w[i] > 0.0f) {
        const float z = (float)x[at[i]] * inv_t;
        part = z == -INFINITY && lse == lse ? INFINITY : w[i] * (lw[i] - (z - lse));
      }
    }
    part = block_all(part, red, [](float a, float b) { return a + b; });
    if (i == 0) {
      p.loss[r] = part * (p.in.temperature * p.in.temperature);
      if (p.lse) p.lse[r] = lse;
    }
    __syncthreads();
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) distill_backward_kernel(DistillDesc p, float inv_t) {
  __shared__ float red[kThreads / 64], w[kTeacherMax], lw[kTeacherMax];
  __shared__ int64_t at[kTeacherMax];
  for (long r = blockIdx.x; r < p.in.rows; r += gridDim.x) {
    const T *x = static_cast<const T *>(p.in.x) + r * p.in.ld;
    T *g = static_cast<T *>(p.grad) + r * p.ldg;
    const bool some = teacher_row(p, r, inv_t, w, lw, at, red);
    const float lse = p.lse_in[r], gt = p.grad_loss[r] * p.in.temperature;
    const bool none = !some || gt == 0.0f;
    const float bad = some && w[0] != w[0] ? NAN : 0.0f;
    // The entries' logits are read before anything of the row is written (grad may be the logits).
    float mine = 0.0f;
    const int i = threadIdx.x;
    const long id = some && i < p.k ? at[i] : -1;
    if (id >= 0 && !none) {
      float sum = 0.0f;  // an id may occur more than once: all of its occurrences write the same value
      for (int j = 0; j < p.k; ++j) sum += at[j] == id ? w[j] : 0.0f;
      const float q = lse == -INFINITY ? 0.0f : expf((float)x[id] * inv_t - lse);
      mine = gt * (q - sum + bad);
    }
    __syncthreads();
    for (long c = threadIdx.x; c < p.in.cols; c += kThreads) {
      const float q = lse == -INFINITY ? 0.0f : expf((float)x[c] * inv_t - lse);
      g[c] = (T)(none ? 0.0f : gt * (q + bad));
    }
    __syncthreads();
    if (id >= 0 && !none) g[id] = (T)mine;
    __syncthreads();
  }
}

// ------------------------------------------------------------------ host
int check_logits(const char *what, const LogitsDesc &d, CError *err) {
  size_t n;
  if (d.dtype != GN_F32 && d.dtype != GN_F16) return set_error(err, -1, "%s: unsupported dtype %d", what, d.dtype);
  if (d.rows < 0 || d.cols < 1 || d.cols > INT_MAX)
    return set_error(err, -1, "%s: invalid size %ld x %ld", what, d.rows, d.cols);
  if (!(d.temperature > 0.0f) || !(1.0f / d.temperature > 0.0f) || !(1.0f / d.temperature < INFINITY))
    return set_error(err, -1, "%s: a temperature above 0 and finite, with a finite reciprocal, is needed", what);
  if (d.ld < d.cols) return set_error(err, -1, "%s: leading dimension %ld smaller than row length %ld", what, d.ld, d.cols);
  if (!matrix_bytes(d.rows, d.ld, 4, &n) || n > ((size_t)1 << 62)) return set_error(err, -1, "%s: too large", what);
  if (d.rows == 0) return 0;
  if (!d.x) return set_error(err, -1, "%s: NULL logits", what);
  if ((uintptr_t)d.x % (d.dtype == GN_F16 ? 2 : 4)) return set_error(err, -1, "%s: logits not aligned to their type", what);
  return 0;
}

int check_workspace(const char *what, const LogitsDesc &d, int k, const void *ws, size_t bytes, CError *err) {
  const size_t need = logits_workspace(d.rows, d.cols, k);
  if (need == 0) return 0;
  if (!ws || bytes < need) return set_error(err, -1, "%s: a workspace of %zu bytes is needed, got %zu", what, need, ws ? bytes : 0);
  if ((uintptr_t)ws % 16) return set_error(err, -1, "%s: a workspace at a multiple of 16 bytes is needed", what);
  return 0;
}

int check_grad(const char *what, const LogitsDesc &d, const void *grad, long ldg, CError *err) {
  size_t n;
  if (ldg < d.cols) return set_error(err, -1, "%s: leading dimension %ld of the gradient smaller than row length %ld", what, ldg, d.cols);
  if (!matrix_bytes(d.rows, ldg, 4, &n) || n > ((size_t)1 << 62)) return set_error(err, -1, "%s: too large", what);
  if (d.rows == 0) return 0;
  if (!grad) return set_error(err, -1, "%s: NULL gradient", what);
  if ((uintptr_t)grad % (d.dtype == GN_F16 ? 2 : 4)) return set_error(err, -1, "%s: gradient not aligned to its type", what);
  if (grad == d.x && ldg != d.ld) return set_error(err, -1, "%s: a gradient in place needs the logits' leading dimension", what);
  return 0;
}

int launched(const char *what, CError *err) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : hip_error(err, -6, what, e);
}

unsigned row_grid(long rows) { return (unsigned)std::min(rows, 1L << 20); }

}  // namespace

size_t logits_workspace(long rows, long cols, int k) {
  (void)rows, (void)cols, (void)k;
  return 0;
}

int check_token_logprobs(const LogprobsDesc &d, CError *err) {
  const char *what = "token logprobs";
  if (int rc = check_logits(what, d.in, err)) return rc;
  if (d.k < 0 || d.k > kTopMax || d.k > d.in.cols)
    return set_error(err, -1, "%s: 0 to %ld alternatives, got %d", what, std::min<long>(kTopMax, d.in.cols), d.k);
  if (d.in.rows == 0) return 0;
  if (!d.targets != !d.logprob) return set_error(err, -1, "%s: targets and logprob are given together", what);
  if (d.k > 0 && (!d.top_ids || !d.top_logprobs)) return set_error(err, -1, "%s: NULL top_ids or top_logprobs", what);
  return check_workspace(what, d.in, d.k, d.workspace, d.workspace_bytes, err);
}

int launch_token_logprobs(const LogprobsDesc &d, hipStream_t s, CError *err) {
  if (d.in.rows == 0) return 0;
  const dim3 grid(row_grid(d.in.rows));
  const float inv_t = 1.0f / d.in.temperature;
  if (d.in.dtype == GN_F16)
    hipLaunchKernelGGL(logprobs_kernel<_Float16>, grid, dim3(kThreads), 0, s, d, inv_t);
  else
    hipLaunchKernelGGL(logprobs_kernel<float>, grid, dim3(kThreads), 0, s, d, inv_t);
  return launched("token logprobs launch", err);
}

int check_token_logprobs_backward(const LogprobsGradDesc &d, CError *err) {
  const char *what = "token logprobs backward";
  if (int rc = check_logits(what, d.in, err)) return rc;
  if (int rc = check_grad(what, d.in, d.grad, d.ldg, err)) return rc;
  if (d.in.rows == 0) return 0;
  if (!d.lse) return set_error(err, -1, "%s: NULL lse", what);
  if (!d.targets != !d.grad_logprob) return set_error(err, -1, "%s: targets and grad_logprob are given together", what);
  if (!d.entropy != !d.grad_entropy) return set_error(err, -1, "%s: entropy and grad_entropy are given together", what);
  return 0;
}

int launch_token_logprobs_backward(const LogprobsGradDesc &d, hipStream_t s, CError *err) {
  if (d.in.rows == 0) return 0;
  const dim3 grid(row_grid(d.in.rows));
  const float inv_t = 1.0f / d.in.temperature;
  if (d.in.dtype == GN_F16)
    hipLaunchKernelGGL(logprobs_backward_kernel<_Float16>, grid, dim3(kThreads), 0, s, d, inv_t);
  else
    hipLaunchKernelGGL(logprobs_backward_kernel<float>, grid, dim3(kThreads), 0, s, d, inv_t);
  return launched("token logprobs backward launch", err);
}

static int check_distill(const char *what, const DistillDesc &d, CError *err) {
  if (int rc = check_logits(what, d.in, err)) return rc;
  if (d.k < 1 || d.k > kTeacherMax) return set_error(err, -1, "%s: 1 to %d entries to a row, got %d", what, kTeacherMax, d.k);
  if (d.in.rows > 0 && (!d.ids || !d.teacher)) return set_error(err, -1, "%s: NULL ids or teacher logits", what);
  return 0;
}

int check_distill_forward(const DistillDesc &d, CError *err) {
  const char *what = "distill forward";
  if (int rc = check_distill(what, d, err)) return rc;
  if (d.in.rows == 0) return 0;
  if (!d.loss) return set_error(err, -1, "%s: NULL loss", what);
  return check_workspace(what, d.in, 0, d.workspace, d.workspace_bytes, err);
}

int launch_distill_forward(const DistillDesc &d, hipStream_t s, CError *err) {
  if (d.in.rows == 0) return 0;
  const dim3 grid(row_grid(d.in.rows));
  const float inv_t = 1.0f / d.in.temperature;
  if (d.in.dtype == GN_F16)
    hipLaunchKernelGGL(distill_kernel<_Float16>, grid, dim3(kThreads), 0, s, d, inv_t);
  else
    hipLaunchKernelGGL(distill_kernel<float>, grid, dim3(kThreads), 0, s, d, inv_t);
  return launched("distill forward launch", err);
}

int check_distill_backward(const DistillDesc &d, CError *err) {
  const char *what = "distill backward";
  if (int rc = check_distill(what, d, err)) return rc;
  if (int rc = check_grad(what, d.in, d.grad, d.ldg, err)) return rc;
  if (d.in.rows > 0 && (!d.lse_in || !d.grad_loss)) return set_error(err, -1, "%s: NULL lse or grad_loss", what);
  return 0;
}

int launch_distill_backward(const DistillDesc &d, hipStream_t s, CError *err) {
  if (d.in.rows == 0) return 0;
  const dim3 grid(row_grid(d.in.rows));
  const float inv_t = 1.0f / d.in.temperature;
  if (d.in.dtype == GN_F16)
    hipLaunchKernelGGL(distill_backward_kernel<_Float16>, grid, dim3(kThreads), 0, s, d, inv_t);
  else
    hipLaunchKernelGGL(distill_backward_kernel<float>, grid, dim3(kThreads), 0, s, d, inv_t);
  return launched("distill backward launch", err);
}

}  // namespace gn
