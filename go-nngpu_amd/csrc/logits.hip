// logits.hip — rows of logits: log-sum-exp, log-probabilities of given tokens, entropy, the top
// alternatives, distillation from a teacher's top logits, and the gradients of the logits.
//
// With z = x / T, m = max z, s = sum e^(z - m) and t = sum (z - m) e^(z - m): lse = m + ln s and the entropy is
// ln s - t / s, two terms that are never negative (no cancellation). All sums are fp32.
//
// All of it is bound by one pass over the logits (and one over the gradients). A workgroup takes a segment of a
// row, up to 8192 logits, in one go into registers: all loads are in flight together, the maximum is known before the
// first exponential, and the top alternatives are looked for in registers. Rows of several segments leave (m, s, t) and the
// segment's best k in the workspace, and a second kernel, one workgroup to a row, joins them in segment order.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "logits.h"

namespace gn {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kFloor = -200.0f;  // e^x is 0 in fp32 from here down: stands in for -inf where that meets a 0

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));

// ------------------------------------------------------------------ a segment in registers
// 16 bytes at any address that is a multiple of T's size (the hardware takes unaligned vectors).
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Unaligned16 {
  u32x4_t v;
};
template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

__device__ __forceinline__ void unpack(u32x4_t a, float (&v)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(a[j]);
}
__device__ __forceinline__ void unpack(u32x4_t a, float (&v)[8]) {
  const half8_t h = __builtin_bit_cast(half8_t, a);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = (float)h[j];
}

// Value e of a thread is the segment's number position<T>(e).
template <typename T>
__device__ __forceinline__ int position(int e) {
  return (e / kVec<T> * kThreads + (int)threadIdx.x) * kVec<T> + e % kVec<T>;
}

// E values of the `left` at x, -inf past them.
template <typename T, int E>
__device__ __forceinline__ void load_segment(const T *x, int left, float (&v)[E]) {
  constexpr int V = kVec<T>;
#pragma unroll
  for (int i = 0; i < E / V; ++i) {
    const int at = position<T>(i * V);
    float u[V];
    if (at + V <= left) {
      unpack(reinterpret_cast<const Unaligned16<T> *>(x + at)->v, u);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) u[j] = at + j < left ? (float)x[at + j] : -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) v[i * V + j] = u[j];
  }
}

__device__ __forceinline__ u32x4_t pack(const float (&v)[4]) {
  return u32x4_t{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
}
__device__ __forceinline__ u32x4_t pack(const float (&v)[8]) {
  half8_t h;
#pragma unroll
  for (int j = 0; j < 8; ++j) h[j] = (_Float16)v[j];
  return __builtin_bit_cast(u32x4_t, h);
}

template <typename T, int E>
__device__ __forceinline__ void store_segment(T *g, int left, const float (&v)[E]) {
  constexpr int V = kVec<T>;
#pragma unroll
  for (int i = 0; i < E / V; ++i) {
    const int at = position<T>(i * V);
    if (at + V <= left) {
      float u[V];
#pragma unroll
      for (int j = 0; j < V; ++j) u[j] = v[i * V + j];
      reinterpret_cast<Unaligned16<T> *>(g + at)->v = pack(u);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (at + j < left) g[at + j] = (T)v[i * V + j];
    }
  }
}

// ------------------------------------------------------------------ reductions
// Over the workgroup's threads; every thread gets the result. red: one value for each wave.
template <typename T, typename F>
__device__ __forceinline__ T block_all(T v, T *red, F op) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = op(v, __shfl_xor(v, o, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) v = op(v, red[i]);
  return v;
}
__device__ __forceinline__ float block_max(float v, float *red) {
  return block_all(v, red, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float block_sum(float v, float *red) {
  return block_all(v, red, [](float a, float b) { return a + b; });
}

struct RowStats {
  float m, s, t;  // max z; sums of e^(z - m) and (z - m) e^(z - m)
};

// e^d. The argument is rounded once (2^-24 |d| relative in the result), results below 2^-126 are 0.
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }

template <int E>
__device__ __forceinline__ RowStats segment_stats(const float (&x)[E], float inv_t, float *red) {
  RowStats r{-INFINITY, 0.0f, 0.0f};
#pragma unroll
  for (int e = 0; e < E; ++e) r.m = fmaxf(r.m, x[e] * inv_t);
  r.m = block_max(r.m, red);
  const float m = r.m == -INFINITY ? 0.0f : r.m;  // a row of -inf: all terms e^-inf = 0
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float d = x[e] * inv_t - m, p = exp_of(d);
    r.s += p;
    r.t += p * fmaxf(d, kFloor);  // 0 where p is 0 and d is -inf; NaN where p is
  }
  r.s = block_sum(r.s, red);
  r.t = block_sum(r.t, red);
  return r;
}
__device__ __forceinline__ float lse_of(const RowStats &r) { return r.s == 0.0f ? -INFINITY : r.m + logf(r.s); }
__device__ __forceinline__ float entropy_of(const RowStats &r) { return r.s == 0.0f ? 0.0f : logf(r.s) - r.t / r.s; }
__device__ __forceinline__ float logprob_of(float z, float lse) { return lse == -INFINITY ? -INFINITY : z - lse; }

// a and b as of one row (b the later segment).
__device__ __forceinline__ RowStats join_stats(const RowStats &a, const RowStats &b) {
  const float m = fmaxf(a.m, b.m), n = m == -INFINITY ? 0.0f : m;
  const float da = fmaxf(a.m - n, kFloor), db = fmaxf(b.m - n, kFloor);  // a segment of -inf has s = t = 0
  const float ea = exp_of(da), eb = exp_of(db);
  RowStats r{m, a.s * ea + b.s * eb, 0.0f};
  r.t = (a.s == 0.0f ? 0.0f : ea * (a.t + da * a.s)) + (b.s == 0.0f ? 0.0f : eb * (b.t + db * b.s));
  // A NaN among the logits is in s, and so is +inf (inf - inf); m does not show NaN.
  return r;
}

// ------------------------------------------------------------------ the top alternatives
// Their order is the larger value first, then the lower column. A float's bits as an unsigned number that is ordered as
// the values are (NaN above infinity, -0 as 0), and with the column below it a key of its own for each entry. 0: no entry
// (of a float, only a negative NaN would have it).
__device__ __forceinline__ uint32_t value_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  if ((b & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  if (k == 0xffffffffu) return NAN;
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ uint64_t entry_key(uint32_t value, uint32_t col) { return ((uint64_t)value << 32) | ~col; }

// The k-th largest of the wave's 64 values (k >= 1), bit by bit: the largest number that k lanes reach.
__device__ __forceinline__ uint32_t wave_kth(uint32_t v, int k) {
  uint32_t t = 0;
#pragma unroll
  for (int b = 31; b >= 0; --b) {
    const uint32_t c = t | (1u << b);
    if (__popcll(__ballot(v >= c)) >= k) t = c;
  }
  return t;
}

constexpr int kCandidates = 1024;

struct TopShared {
  uint64_t key[kCandidates], bound[kWaves];
  int count;
};

// Writes the k largest of n keys in sh.key to out, in order; 0 where there are fewer. Each key's place is the number of
// larger ones (no two are equal).
__device__ __forceinline__ void write_ranked(const TopShared &sh, int n, int k, uint64_t *out) {
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const uint64_t mine = sh.key[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += sh.key[j] > mine;
    if (rank < k) out[rank] = mine;
  }
  for (int i = n + threadIdx.x; i < k; i += kThreads) out[i] = 0;
}

// The k largest entries of a segment, in order, to out (LDS or memory). The k-th largest of a wave's 64 lane maxima bounds
// its own k-th largest value from below, the largest of the waves' bounds the segment's; what reaches that (some 4 k values of
// 8192 in no particular order) is gathered in LDS and ranked. The bound is a whole key, so equal values do not all
// reach it: at most k entries to a lane and wave do. Where they are too many all the same (large values side by side
// in few lanes), the best is looked for k times.
template <typename T, int E>
__device__ __forceinline__ void segment_top(const float (&x)[E], int left, uint32_t col0, int k, TopShared &sh, uint64_t *out) {
  uint32_t best = 0, best_col = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int at = position<T>(e);
    const uint32_t v = at < left ? value_key(x[e]) : 0;
    if (v > best) best = v, best_col = at;  // a lane's columns go up with e
  }
  const uint32_t bound = wave_kth(best, k);
  uint64_t key = entry_key(bound, 0xffffffffu);  // all entries of that value, or with several lanes there the best of them
  const int above = __popcll(__ballot(best > bound)), equal = __popcll(__ballot(best == bound));
  if (bound != 0 && above + equal > k) key = entry_key(bound, 0) & ~0xffffffffull | wave_kth(best == bound ? ~(col0 + best_col) : 0, k - above);
  if ((threadIdx.x & 63) == 0) sh.bound[threadIdx.x >> 6] = bound ? key : 1;
  if (threadIdx.x == 0) sh.count = 0;
  __syncthreads();
  key = sh.bound[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) key = max(key, sh.bound[i]);
  const uint32_t key_value = (uint32_t)(key >> 32);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int at = position<T>(e);
    const uint32_t v = value_key(x[e]);
    if (v >= key_value && at < left) {
      const uint64_t c = entry_key(v, col0 + at);
      if (c >= key) {
        const int i = atomicAdd(&sh.count, 1);  // the places' order changes nothing: they are ranked
        if (i < kCandidates) sh.key[i] = c;
      }
    }
  }
  __syncthreads();
  const int n = sh.count;
  if (n <= kCandidates) {
    write_ranked(sh, n, k, out);
  } else {
    uint64_t last = ~0ull;
    for (int i = 0; i < k; ++i) {
      uint64_t mine = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int at = position<T>(e);
        const uint64_t c = at < left ? entry_key(value_key(x[e]), col0 + at) : 0;
        if (c < last && c > mine) mine = c;
      }
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) mine = max(mine, (uint64_t)__shfl_xor((unsigned long long)mine, o, 64));
      __syncthreads();
      if ((threadIdx.x & 63) == 0) sh.bound[threadIdx.x >> 6] = mine;
      __syncthreads();
      last = sh.bound[0];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) last = max(last, sh.bound[w]);
      if (threadIdx.x == 0) out[i] = last;
    }
  }
  __syncthreads();
}

// ------------------------------------------------------------------ a row's results
template <typename T>
__device__ __forceinline__ void finish_logprobs(const LogprobsDesc &p, long r, const RowStats &st, const uint64_t *top, float inv_t) {
  const float lse = lse_of(st);
  if (threadIdx.x == 0) {
    if (p.lse) p.lse[r] = lse;
    if (p.entropy) p.entropy[r] = entropy_of(st);
    if (p.targets) {
      const long t = p.targets[r];
      const T *x = static_cast<const T *>(p.in.x) + r * p.in.ld;
      p.logprob[r] = t < 0 ? 0.0f : t >= p.in.cols ? NAN : logprob_of((float)x[t] * inv_t, lse);
    }
  }
  if ((int)threadIdx.x < p.k) {
    const uint64_t key = top[threadIdx.x];
    p.top_ids[r * p.k + threadIdx.x] = (int64_t)(uint32_t)~key;
    p.top_logprobs[r * p.k + threadIdx.x] = logprob_of(key_value((uint32_t)(key >> 32)) * inv_t, lse);
  }
}

// The teacher's distribution over its k entries: w, its logarithm lw, the columns at (-1, and w = 0, for absent ones).
// Returns false for a row without entries; w is NaN throughout where an id is too large or a logit is NaN or +inf.
struct Teacher {
  float w[kTeacherMax], lw[kTeacherMax];
  int at[kTeacherMax];
  float red[kWaves];
};
__device__ __forceinline__ bool teacher_row(const DistillDesc &p, long r, float inv_t, Teacher &sh) {
  const int i = threadIdx.x;
  int at = -1;
  float z = -INFINITY;
  if (i < p.k) {
    const int64_t id = p.ids[r * p.k + i];
    const float t = p.teacher[r * p.k + i];
    if (id >= p.in.cols)
      z = NAN;
    else if (id >= 0)
      z = t * inv_t, at = (int)id;
    if (z == -INFINITY) at = -1;
  }
  const float m = block_all(z, sh.red, [](float a, float b) { return a != a || b != b ? NAN : fmaxf(a, b); });
  if (m == -INFINITY) return false;
  const float e = z == -INFINITY ? 0.0f : expf(z - m);
  const float s = block_sum(e, sh.red);
  if (i < p.k) {
    sh.w[i] = e / s;
    sh.lw[i] = z - m - logf(s);
    sh.at[i] = at;
  }
  __syncthreads();
  return true;
}

template <typename T>
__device__ __forceinline__ void finish_distill(const DistillDesc &p, long r, const RowStats &st, float inv_t, Teacher &sh) {
  const float lse = lse_of(st);
  const bool some = teacher_row(p, r, inv_t, sh);
  const int i = threadIdx.x;
  float part = 0.0f;
  if (some && i < p.k) {
    if (sh.w[i] != sh.w[i]) {
      part = NAN;
    } else if (sh.at[i] >= 0 && sh.w[i] > 0.0f) {
      const float z = (float)(static_cast<const T *>(p.in.x) + r * p.in.ld)[sh.at[i]] * inv_t;
      part = z == -INFINITY && lse == lse ? INFINITY : sh.w[i] * (sh.lw[i] - (z - lse));
    }
  }
  part = block_sum(part, sh.red);
  if (i == 0) {
    p.loss[r] = part * (p.in.temperature * p.in.temperature);
    if (p.lse) p.lse[r] = lse;
  }
}

// ------------------------------------------------------------------ forward kernels
// The workspace: for each row and segment (row major) its statistics, then for each its k best keys.
struct Work {
  RowStats *stats;
  uint64_t *keys;
};
__host__ __device__ inline size_t stats_bytes(long rows, long segs) { return ((size_t)rows * segs * sizeof(RowStats) + 15) / 16 * 16; }
__host__ __device__ inline Work work_of(void *ws, long rows, long segs) {
  return {static_cast<RowStats *>(ws), reinterpret_cast<uint64_t *>(static_cast<char *>(ws) + stats_bytes(rows, segs))};
}

// D is LogprobsDesc or DistillDesc. TOP: with alternatives. ONE: rows of one segment, finished here.
template <typename T, int E, typename D, bool TOP, bool ONE>
__global__ void __launch_bounds__(kThreads) segment_kernel(D p, float inv_t, int segs) {
  constexpr bool DISTILL = std::is_same_v<D, DistillDesc>;
  __shared__ float red[kWaves];
  __shared__ std::conditional_t<TOP, TopShared, int> top;
  __shared__ uint64_t best[TOP && ONE ? kTopMax : 1];
  __shared__ std::conditional_t<DISTILL && ONE, Teacher, int> teacher;
  const long r = blockIdx.x / segs;
  const int seg = blockIdx.x % segs;
  const long col0 = (long)seg * kThreads * E;
  const int left = (int)min(p.in.cols - col0, (long)kThreads * E);
  float x[E];
  load_segment<T, E>(static_cast<const T *>(p.in.x) + r * p.in.ld + col0, left, x);
  const RowStats st = segment_stats<E>(x, inv_t, red);
  const Work w = work_of(p.workspace, p.in.rows, segs);
  if constexpr (TOP) segment_top<T, E>(x, left, (uint32_t)col0, p.k, top, ONE ? best : w.keys + (r * segs + seg) * p.k);
  if constexpr (ONE) {
    if constexpr (DISTILL)
      finish_distill<T>(p, r, st, inv_t, teacher);
    else
      finish_logprobs<T>(p, r, st, best, inv_t);
  } else if (threadIdx.x == 0) {
    w.stats[r * segs + seg] = st;
  }
}

template <typename T, typename D>
__global__ void __launch_bounds__(kThreads) join_kernel(D p, float inv_t, int segs) {
  constexpr bool DISTILL = std::is_same_v<D, DistillDesc>;
  __shared__ std::conditional_t<DISTILL, Teacher, TopShared> sh;
  __shared__ uint64_t best[kTopMax];
  __shared__ RowStats part[kWaves];
  const long r = blockIdx.x;
  const Work w = work_of(p.workspace, p.in.rows, segs);
  // Each thread its segments in order, then the threads in pairs: an order that depends on the sizes alone.
  RowStats st{-INFINITY, 0.0f, 0.0f};
  for (int i = threadIdx.x; i < segs; i += kThreads) st = join_stats(st, w.stats[r * segs + i]);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const RowStats b{__shfl_xor(st.m, o, 64), __shfl_xor(st.s, o, 64), __shfl_xor(st.t, o, 64)};
    st = threadIdx.x & o ? join_stats(b, st) : join_stats(st, b);
  }
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = st;
  __syncthreads();
  st = part[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) st = join_stats(st, part[i]);
  if constexpr (DISTILL) {
    finish_distill<T>(p, r, st, inv_t, sh);
  } else {
    if (p.k > 0) {
      // Every segment's k are in order: the largest of their last ones bounds the row's k-th from below. What reaches it is
      // ranked, a part of the segments at a time where they are more than there is room for (with the best so far).
      const uint64_t *keys = w.keys + r * segs * p.k;
      const int k = p.k, group = kCandidates / k - 1;
      int kept = 0;
      for (int s0 = 0; s0 < segs; s0 += group) {
        const int count = min(group, segs - s0);
        if (threadIdx.x == 0) sh.count = kept;
        uint64_t bound = 1;
        for (int i = threadIdx.x; i < count; i += kThreads) bound = max(bound, keys[(long)(s0 + i) * k + k - 1]);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) bound = max(bound, (uint64_t)__shfl_xor((unsigned long long)bound, o, 64));
        if ((threadIdx.x & 63) == 0) sh.bound[threadIdx.x >> 6] = bound;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kWaves; ++i) bound = max(bound, sh.bound[i]);
        for (int i = threadIdx.x; i < kept; i += kThreads) sh.key[i] = best[i];
        for (int i = threadIdx.x; i < count * k; i += kThreads) {
          const uint64_t c = keys[(long)s0 * k + i];
          if (c >= bound) sh.key[atomicAdd(&sh.count, 1)] = c;  // ranked, whatever the places' order
        }
        __syncthreads();
        const int n = sh.count;
        write_ranked(sh, n, k, best);
        kept = min(n, k);
        __syncthreads();
      }
    }
    finish_logprobs<T>(p, r, st, best, inv_t);
  }
}

// ------------------------------------------------------------------ backward kernels
// A workgroup to a segment, as in the forward pass: one read and one write. A row whose gradient is 0 is not read.
template <typename T, int E>
__global__ void __launch_bounds__(kThreads) logprobs_backward_kernel(LogprobsGradDesc p, float inv_t, int segs) {
  const long r = blockIdx.x / segs, col0 = (long)(blockIdx.x % segs) * kThreads * E;
  const int left = (int)min(p.in.cols - col0, (long)kThreads * E);
  const long t = p.targets ? p.targets[r] : -1;
  const float lse = p.lse[r], gh = p.grad_entropy ? p.grad_entropy[r] : 0.0f, h = p.grad_entropy ? p.entropy[r] : 0.0f;
  float gl = t >= 0 ? p.grad_logprob[r] : 0.0f;
  if (t >= p.in.cols) gl = NAN;
  const bool none = (gl == 0.0f && gh == 0.0f) || (lse == -INFINITY && t < p.in.cols);
  float x[E];
  if (none) {
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = 0.0f;
  } else {
    load_segment<T, E>(static_cast<const T *>(p.in.x) + r * p.in.ld + col0, left, x);
    const int at = t >= col0 && t < col0 + left ? (int)(t - col0) : -1;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float lp = x[e] * inv_t - lse, q = exp_of(lp);
      float v = -q * (gl + gh * (fmaxf(lp, kFloor) + h));  // 0 where q is 0 and lp is -inf
      if (position<T>(e) == at) v += gl;
      x[e] = v * inv_t;
    }
  }
  store_segment<T, E>(static_cast<T *>(p.grad) + r * p.ldg + col0, left, x);
}

template <typename T, int E>
__global__ void __launch_bounds__(kThreads) distill_backward_kernel(DistillDesc p, float inv_t, int segs) {
  __shared__ Teacher sh;
  const long r = blockIdx.x / segs, col0 = (long)(blockIdx.x % segs) * kThreads * E;
  const int left = (int)min(p.in.cols - col0, (long)kThreads * E);
  const T *row = static_cast<const T *>(p.in.x) + r * p.in.ld + col0;
  T *out = static_cast<T *>(p.grad) + r * p.ldg + col0;
  const float lse = p.lse_in[r], gt = p.grad_loss[r] * p.in.temperature;
  float x[E];
  if (gt != 0.0f) load_segment<T, E>(row, left, x);
  const bool some = teacher_row(p, r, inv_t, sh);
  const bool none = !some || gt == 0.0f;
  const float bad = some && sh.w[0] != sh.w[0] ? NAN : 0.0f;
  // The entries of this segment are put right once the segment is written; their logits are read before (grad may be
  // the logits). An id may occur more than once: all of its occurrences write the same value.
  const int i = threadIdx.x;
  const long at = some && i < p.k ? sh.at[i] - col0 : -1;
  const bool mine = !none && at >= 0 && at < left;
  float fix = 0.0f;
  if (mine) {
    float sum = 0.0f;
    for (int j = 0; j < p.k; ++j) sum += sh.at[j] == sh.at[i] ? sh.w[j] : 0.0f;
    fix = gt * ((lse == -INFINITY ? 0.0f : exp_of((float)row[at] * inv_t - lse)) - sum + bad);
  }
  const bool any = __syncthreads_or(mine);
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = none ? 0.0f : gt * ((lse == -INFINITY ? 0.0f : exp_of(x[e] * inv_t - lse)) + bad);
  store_segment<T, E>(out, left, x);
  if (any) {
    __syncthreads();
    if (mine) out[at] = (T)fix;
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
  // A workgroup to 2048 columns and more of a row, below 2^24 of them (2^32 threads).
  if (!matrix_bytes(d.rows, d.ld, 4, &n) || n > ((size_t)1 << 62) || d.rows >= (1L << 24) / ((d.cols + 8191) / 8192))
    return set_error(err, -1, "%s: %ld x %ld is too large", what, d.rows, d.cols);
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

// Values of a row to a thread: 32, 8192 logits to a workgroup, or 8 where that leaves CUs without one (one row of
// 131072, 20 alternatives: 16 workgroups of 8192 take TBD us, 64 of 2048 TBD).
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

template <typename D>
int launch_forward(const D &d, const char *what, hipStream_t s, CError *err) {
  constexpr bool DISTILL = std::is_same_v<D, DistillDesc>;
  const Split sp = split_of(d.in.rows, d.in.cols);
  const dim3 grid((unsigned)(d.in.rows * sp.segs)), block(kThreads);
  const float inv_t = 1.0f / d.in.temperature;
  with_kind(d.in.dtype, sp.per, [&](auto type, auto per) {
    using T = decltype(type);
    constexpr int E = decltype(per)::value;
    auto launch = [&](auto top) {
      constexpr bool TOP = decltype(top)::value;
      if (sp.segs == 1) {
        hipLaunchKernelGGL((segment_kernel<T, E, D, TOP, true>), grid, block, 0, s, d, inv_t, 1);
      } else {
        hipLaunchKernelGGL((segment_kernel<T, E, D, TOP, false>), grid, block, 0, s, d, inv_t, sp.segs);
        hipLaunchKernelGGL((join_kernel<T, D>), dim3((unsigned)d.in.rows), block, 0, s, d, inv_t, sp.segs);
      }
    };
    if constexpr (DISTILL) {
      launch(std::false_type{});
    } else {
      if (d.k > 0)
        launch(std::true_type{});
      else
        launch(std::false_type{});
    }
  });
  return launched(what, err);
}

}  // namespace

size_t logits_workspace(long rows, long cols, int k) {
  if (rows < 1 || cols < 1 || k < 0) return 0;
  const Split sp = split_of(rows, cols);
  if (sp.segs == 1) return 0;
  return stats_bytes(rows, sp.segs) + (size_t)rows * sp.segs * k * sizeof(uint64_t);
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
  return d.in.rows == 0 ? 0 : launch_forward(d, "token logprobs launch", s, err);
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
  const Split sp = split_of(d.in.rows, d.in.cols);
  const dim3 grid((unsigned)(d.in.rows * sp.segs));
  with_kind(d.in.dtype, sp.per, [&](auto type, auto per) {
    hipLaunchKernelGGL((logprobs_backward_kernel<decltype(type), decltype(per)::value>), grid, dim3(kThreads), 0, s, d,
                       1.0f / d.in.temperature, sp.segs);
  });
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
  return d.in.rows == 0 ? 0 : launch_forward(d, "distill forward launch", s, err);
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
  const Split sp = split_of(d.in.rows, d.in.cols);
  const dim3 grid((unsigned)(d.in.rows * sp.segs));
  with_kind(d.in.dtype, sp.per, [&](auto type, auto per) {
    hipLaunchKernelGGL((distill_backward_kernel<decltype(type), decltype(per)::value>), grid, dim3(kThreads), 0, s, d,
                       1.0f / d.in.temperature, sp.segs);
  });
  return launched("distill backward launch", err);
}

}  // namespace gn
