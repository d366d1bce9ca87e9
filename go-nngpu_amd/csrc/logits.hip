// logits.hip — rows of logits: log-sum-exp, log-probabilities of given tokens, entropy, the top
// alternatives, distillation from a teacher's top logits, and the gradients of the logits.
//
// With z = x / T, m = max z, s = sum e^(z - m) and t = sum (z - m) e^(z - m): lse = m + ln s and the entropy is
// ln s - t / s, two terms that are never negative (no cancellation). All sums are fp32. Exponents are taken in base 2, of
// (x - max x) c with the rounded c = log2(e) / T.
//
// All of it is bound by one pass over the logits (and one over the gradients). A workgroup takes a segment of a
// row, up to 8192 logits, in one go into registers: all loads are in flight together, the maximum is known before the
// first exponential, and the top alternatives are looked for in registers. Rows of several segments leave (m, s, t) and the
// segment's best k in the workspace, and a second kernel, one workgroup to a row, joins them in segment order.
// Measured (a large copy 4.6, reads alone 5.4 TB/s): 4096 rows of 32768 in fp32 103 us forward (5.2 TB/s), 180 with 20
// alternatives (141 registers against 92 leave 3 waves to a SIMD instead of 5, for the loads as for the search), 191 backward (5.6);
// distillation of 2048 rows of 65536 in fp16 54 us forward, 96 backward (5.6). One row of 131072 takes 5.8 us, the
// latencies of two launches and their reductions, and with 20 alternatives 12.8: those of the two searches too.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "logits.h"

namespace gn {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr float kFloor = -300.0f;  // 2^x is 0 in fp32 from here down: stands in for -inf where that meets a 0

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------ a segment in registers
// 16 bytes at any address that is a multiple of T's size (the hardware takes unaligned vectors).
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Unaligned16 {
  u32x4_t v;
};
template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

// Value e of a thread is the segment's number position<T>(e).
template <typename T>
__device__ __forceinline__ int position(int e) {
  return (e / kVec<T> * kThreads + (int)threadIdx.x) * kVec<T> + e % kVec<T>;
}

// A thread's E values of a segment, in their own type.
template <typename T, int E>
struct Segment {
  typedef T V __attribute__((ext_vector_type(kVec<T>)));
  V v[E / kVec<T>];
  __device__ __forceinline__ float operator[](int e) const { return (float)v[e / kVec<T>][e % kVec<T>]; }

  // The `left` values at x, -inf past them.
  __device__ __forceinline__ void load(const T *x, int left) {
#pragma unroll
    for (int i = 0; i < E / kVec<T>; ++i) {
      const int at = position<T>(i * kVec<T>);
      if (at + kVec<T> <= left) {
        v[i] = __builtin_bit_cast(V, reinterpret_cast<const Unaligned16<T> *>(x + at)->v);
      } else {
#pragma unroll
        for (int j = 0; j < kVec<T>; ++j) v[i][j] = at + j < left ? x[at + j] : (T)-INFINITY;
      }
    }
  }
  __device__ __forceinline__ void store(T *g, int left) const {
#pragma unroll
    for (int i = 0; i < E / kVec<T>; ++i) {
      const int at = position<T>(i * kVec<T>);
      if (at + kVec<T> <= left) {
        reinterpret_cast<Unaligned16<T> *>(g + at)->v = __builtin_bit_cast(u32x4_t, v[i]);
      } else {
#pragma unroll
        for (int j = 0; j < kVec<T>; ++j)
          if (at + j < left) g[at + j] = v[i][j];
      }
    }
  }
  // Of the numbers among them (fp16: two to an instruction), -inf without any.
  __device__ __forceinline__ float max_value() const {
    V m = v[0];
#pragma unroll
    for (int i = 1; i < E / kVec<T>; ++i) m = __builtin_elementwise_max(m, v[i]);
    float r = -INFINITY;
#pragma unroll
    for (int j = 0; j < kVec<T>; ++j) r = fmaxf(r, (float)m[j]);
    return r;
  }
};

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

// m: the largest x; s: the sum of 2^d, d = (x - m) c; t: that of d 2^d.
struct RowStats {
  float m, s, t;
};

__device__ __forceinline__ float exp2_of(float d) { return __builtin_amdgcn_exp2f(d); }  // results below 2^-126 are 0

// largest: the thread's largest value. T: with t.
template <bool T, typename S, int E>
__device__ __forceinline__ RowStats segment_stats(const Segment<S, E> &x, float largest, float c, float *red) {
  RowStats r{block_max(largest, red), 0.0f, 0.0f};
  const float m = r.m == -INFINITY ? 0.0f : r.m;  // a segment of -inf: all terms 2^-inf = 0
  const float mc = m * c;
  // fp16: one fma, as it is bound by its instructions, each d too large by what rounding m c lost (at most 1/4); not where m c is
  // large, nor in fp32, whose lowest value times c would be -inf.
  auto terms = [&](auto fused) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float d = decltype(fused)::value ? fmaf(x[e], c, -mc) : (x[e] - m) * c, p = exp2_of(d);
      r.s += p;
      if (T) r.t += p * fmaxf(d, kFloor);  // 0 where p is 0 and d is -inf; NaN where p is
    }
  };
  const bool fused = sizeof(S) == 2 && fabsf(mc) <= 0x1p22f;  // the same in all threads
  if (fused)
    terms(std::true_type{});
  else
    terms(std::false_type{});
  r.s = block_sum(r.s, red);
  if (T) r.t = block_sum(r.t, red);
  if (fused) {
    const float lost = fmaf(m, c, -mc);
    r.s *= exp2_of(-lost);
    if (T) r.t = r.t * exp2_of(-lost) - lost * r.s;
  }
  return r;
}
__device__ __forceinline__ float lse_of(const RowStats &r, float inv_t) {
  return r.s == 0.0f ? -INFINITY : fmaf(r.m, inv_t, log2f(r.s) * kLn2);
}
__device__ __forceinline__ float entropy_of(const RowStats &r) { return r.s == 0.0f ? 0.0f : (log2f(r.s) - r.t / r.s) * kLn2; }
// Of x, from its distance to the maximum: lse may be too large to hold ln s beside it.
__device__ __forceinline__ float logprob_of(float x, const RowStats &r, float inv_t) {
  return r.s == 0.0f ? -INFINITY : fmaf(x - r.m, inv_t, -log2f(r.s) * kLn2);
}

// The statistics of the row that the threads' segments make up, each thread's in an order that the sizes alone
// give.
__device__ __forceinline__ RowStats join_stats(const RowStats *stats, int segs, float c, float *red) {
  float m = -INFINITY;
  for (int i = threadIdx.x; i < segs; i += kThreads) m = fmaxf(m, stats[i].m);
  RowStats r{block_max(m, red), 0.0f, 0.0f};
  const float n = r.m == -INFINITY ? 0.0f : r.m;
  for (int i = threadIdx.x; i < segs; i += kThreads) {
    const RowStats a = stats[i];
    // A NaN among the logits is in s, and so is +inf (inf - inf); m does not show NaN. A segment of -inf has s = t = 0.
    const float d = fmaxf((a.m - n) * c, kFloor), e = exp2_of(d);
    r.s += e * a.s;
    r.t += e * (a.t + d * a.s);
  }
  r.s = block_sum(r.s, red);
  r.t = block_sum(r.t, red);
  return r;
}

// ------------------------------------------------------------------ the top alternatives
// Their order is the larger value first, then the lower column. A float's bits as an unsigned number that is ordered as
// the values are (NaN above infinity, -0 as 0), and with the column below it a key of its own for each entry. 0: no entry
// (of a float, only a negative NaN would have it). NaN's is not the largest word: with column 0's complement, which is, the key
// would be the one that the search for the best starts below.
constexpr uint32_t kNanKey = 0xfffffffeu;
__device__ __forceinline__ uint32_t value_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  if ((b & 0x7fffffffu) > 0x7f800000u) return kNanKey;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  if (k == kNanKey) return NAN;
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ uint64_t entry_key(uint32_t value, uint32_t col) { return ((uint64_t)value << 32) | ~col; }

// A number that at least k of the wave's 64 values reach (k >= 1): exactly k where one is that tells them apart, found bit by
// bit (some 13 of the 32 for logits), else the k-th largest value.
__device__ __forceinline__ uint32_t wave_kth(uint32_t v, int k) {
  uint32_t t = 0;
  for (uint32_t bit = 1u << 31; bit != 0; bit >>= 1) {
    const int n = __popcll(__ballot(v >= (t | bit)));
    if (n >= k) t |= bit;
    if (n == k) break;
  }
  return t;
}

constexpr int kCandidates = 1024;                    // of a segment
constexpr int kJoined = kTopMax * (kTopMax + 1);     // of some segments of a row and the best of those before

template <int N>
struct TopShared {
  uint64_t key[N + 8], bound[kWaves];
  int count;
};

// A key that at least k of the workgroup's values reach (some of its threads have one each, no two equal, 0 none):
// each of the `waves` first waves finds the one that ceil(k / waves) of its own reach, and the smallest of these is reached by
// k. About 1.5 k values of k waves' in no particular order do. 1 where a wave has too few.
__device__ __forceinline__ uint64_t block_bound(uint64_t mine, int k, int waves, uint64_t *bound) {
  const int share = (k + waves - 1) / waves;
  const uint32_t hi = (uint32_t)(mine >> 32), lo = (uint32_t)mine;
  const uint32_t value = wave_kth(hi, share);
  const int above = __popcll(__ballot(hi > value)), equal = __popcll(__ballot(hi == value));
  // All of that value, or where those are too many as many as are wanted by their columns.
  uint64_t key = (uint64_t)value << 32;
  if (value != 0 && above + equal > share) key |= wave_kth(hi == value ? lo : 0, share - above);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) bound[threadIdx.x >> 6] = (int)(threadIdx.x >> 6) < waves ? max(key, (uint64_t)1) : ~0ull;
  __syncthreads();
  key = bound[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) key = min(key, bound[i]);
  return key;
}

// Writes the k largest of n keys to out, in order; 0 where there are fewer. Each key's place is the number of
// larger ones (no two are equal). key has room for 8 more.
__device__ __forceinline__ void write_ranked(uint64_t *key, int n, int k, uint64_t *out) {
  if (threadIdx.x < 8) key[n + threadIdx.x] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const uint64_t mine = key[i];
    int rank = 0;
    for (int j = 0; j < n; j += 8) {
#pragma unroll
      for (int u = 0; u < 8; ++u) rank += key[j + u] > mine;
    }
    if (rank < k) out[rank] = mine;
  }
  for (int i = n + threadIdx.x; i < k; i += kThreads) out[i] = 0;
}

// The k largest entries of a segment, in order, to out (LDS or memory): a bound from the lanes' best entries, which is
// a whole key, so that equal values do not all reach it; what reaches it is gathered in LDS and ranked. Where that is too
// much (large values side by side in few lanes), and among NaN or +inf (numbers false), the best is looked for k times.
template <typename T, int E>
__device__ __forceinline__ void segment_top(const Segment<T, E> &x, float largest, bool numbers, int left, uint32_t col0, int k,
                                            TopShared<kCandidates> &sh, uint64_t *out) {
  int n = kCandidates + 1;
  if (numbers) {
    int at = INT_MAX;  // the lane's first place with its largest value
#pragma unroll
    for (int e = E - 1; e >= 0; --e)
      if (x[e] == largest) at = position<T>(e);
    if (threadIdx.x == 0) sh.count = 0;
    // The waves whose lanes all have an entry, or the first one.
    const int waves = max(1, min(kWaves, left / (64 * kVec<T>)));
    const uint64_t key = block_bound(at < left ? entry_key(value_key(largest), col0 + at) : 0, k, waves, sh.bound);
    const uint32_t value = (uint32_t)(key >> 32);
    const float bound = value ? key_value(value) : -INFINITY;  // a cut between numbers may be no number's key: NaN
    const float least = bound == bound ? bound : -INFINITY;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (x[e] >= least) {
        const int i = position<T>(e);
        const uint64_t c = entry_key(value_key(x[e]), col0 + i);
        if (c >= key && i < left) {
          const int to = atomicAdd(&sh.count, 1);  // the places' order changes nothing: they are ranked
          if (to < kCandidates) sh.key[to] = c;
        }
      }
    }
    __syncthreads();
    n = sh.count;
  }
  if (n <= kCandidates) {
    write_ranked(sh.key, n, k, out);
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

// The k largest of segs lists of k in order (0 past their ends), to best in order: some lists at a time, as many as there is
// room for if all of their entries are kept. The threads hold the lists' first entries, or the largest of several lists' first
// ones, and bound the k-th largest from below.
__device__ __forceinline__ void join_top(const uint64_t *keys, int segs, int k, TopShared<kJoined> &sh, uint64_t *best) {
  const int group = kJoined / k - 1;
  int kept = 0;
  for (int s0 = 0; s0 < segs; s0 += group, keys += (long)group * k) {
    const int lists = min(group, segs - s0), depth = kThreads / lists;  // entries of each list that the threads hold
    constexpr int N = (kJoined + kThreads - 1) / kThreads;
    uint64_t all[N], key = 1;  // all entries: under way while the bound is found
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = threadIdx.x + i * kThreads;
      all[i] = at < lists * k ? keys[at] : 0;
    }
    if (lists * k > kThreads) {  // otherwise all are ranked
      uint64_t mine = 0;
      const int held = depth > 0 ? lists * min(depth, k) : kThreads;
      if (depth == 0) {
        for (int s = threadIdx.x; s < lists; s += kThreads) mine = max(mine, keys[(long)s * k]);
      } else if ((int)threadIdx.x < held) {
        mine = keys[threadIdx.x % lists * k + threadIdx.x / lists];
      }
      key = block_bound(mine, k, max(1, held / 64), sh.bound);
    }
    for (int i = threadIdx.x; i < kept; i += kThreads) sh.key[i] = best[i];
    if (threadIdx.x == 0) sh.count = kept;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (all[i] >= key) sh.key[atomicAdd(&sh.count, 1)] = all[i];  // ranked, whatever the places' order
    __syncthreads();
    kept = min(sh.count, k);
    write_ranked(sh.key, sh.count, k, best);
    __syncthreads();
  }
}

// ------------------------------------------------------------------ a row's results
template <typename T>
__device__ __forceinline__ void finish_logprobs(const LogprobsDesc &p, long r, const RowStats &st, const uint64_t *top, float inv_t) {
  if (threadIdx.x == 0) {
    if (p.lse) p.lse[r] = lse_of(st, inv_t);
    if (p.entropy) p.entropy[r] = entropy_of(st);
    if (p.targets) {
      const long t = p.targets[r];
      const T *x = static_cast<const T *>(p.in.x) + r * p.in.ld;
      p.logprob[r] = t < 0 ? 0.0f : t >= p.in.cols ? NAN : logprob_of((float)x[t], st, inv_t);
    }
  }
  if ((int)threadIdx.x < p.k) {
    const uint64_t key = top[threadIdx.x];
    p.top_ids[r * p.k + threadIdx.x] = (int64_t)(uint32_t)~key;
    p.top_logprobs[r * p.k + threadIdx.x] = logprob_of(key_value((uint32_t)(key >> 32)), st, inv_t);
  }
}

// The teacher's distribution over its k entries: w, its logarithm lw, the columns at (-1, and w = 0, for absent ones).
// Returns false for a row without entries; w is NaN throughout where an id is too large or a logit is NaN or +inf.
struct Teacher {
  float w[kTeacherMax], lw[kTeacherMax];
  int at[kTeacherMax];
  float red[kWaves];
};
struct Entry {
  int64_t id;
  float logit;
};
__device__ __forceinline__ Entry load_entry(const DistillDesc &p, long r) {
  const int i = threadIdx.x;
  return i < p.k ? Entry{p.ids[r * p.k + i], p.teacher[r * p.k + i]} : Entry{-1, 0.0f};
}
__device__ __forceinline__ bool teacher_row(const DistillDesc &p, const Entry &entry, float inv_t, Teacher &sh) {
  const int i = threadIdx.x;
  int at = -1;
  float x = -INFINITY;
  if (entry.id >= p.in.cols)
    x = NAN;
  else if (entry.id >= 0)
    x = entry.logit, at = (int)entry.id;
  if (x == -INFINITY) at = -1;
  const float m = block_all(x, sh.red, [](float a, float b) { return a != a || b != b ? NAN : fmaxf(a, b); });
  if (m == -INFINITY) return false;
  const float z = (x - m) * inv_t;
  const float e = expf(z);
  const float s = block_sum(e, sh.red);
  if (i < p.k) {
    sh.w[i] = e / s;
    sh.lw[i] = z - logf(s);
    sh.at[i] = at;
  }
  __syncthreads();
  return true;
}

template <typename T>
__device__ __forceinline__ void finish_distill(const DistillDesc &p, long r, const RowStats &st, float inv_t, Teacher &sh) {
  const bool some = teacher_row(p, load_entry(p, r), inv_t, sh);
  const int i = threadIdx.x;
  float part = 0.0f;
  if (some && i < p.k) {
    if (sh.w[i] != sh.w[i]) {
      part = NAN;
    } else if (sh.at[i] >= 0) {
      const float x = (float)(static_cast<const T *>(p.in.x) + r * p.in.ld)[sh.at[i]];
      if (sh.w[i] > 0.0f)
        part = sh.w[i] * (sh.lw[i] - logprob_of(x, st, inv_t));  // +inf where x is -inf
      else if (x == -INFINITY)
        part = INFINITY;  // p is above 0, if below what fp32 holds
    }
  }
  part = block_sum(part, sh.red);
  if (i == 0) {
    p.loss[r] = part * p.in.temperature * p.in.temperature;
    if (p.lse) p.lse[r] = lse_of(st, inv_t);
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
  __shared__ std::conditional_t<TOP, TopShared<kCandidates>, int> top;
  __shared__ uint64_t best[TOP && ONE ? kTopMax : 1];
  __shared__ std::conditional_t<DISTILL && ONE, Teacher, int> teacher;
  const long r = blockIdx.x / segs;
  const int seg = blockIdx.x % segs;
  const long col0 = (long)seg * kThreads * E;
  const int left = (int)min(p.in.cols - col0, (long)kThreads * E);
  Segment<T, E> x;
  x.load(static_cast<const T *>(p.in.x) + r * p.in.ld + col0, left);
  const float largest = x.max_value();
  const RowStats st = segment_stats<!DISTILL>(x, largest, inv_t * kLog2e, red);
  const Work w = work_of(p.workspace, p.in.rows, segs);
  if constexpr (TOP) segment_top(x, largest, st.s == st.s, left, (uint32_t)col0, p.k, top, ONE ? best : w.keys + (r * segs + seg) * p.k);
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
  __shared__ std::conditional_t<DISTILL, Teacher, TopShared<kJoined>> sh;
  __shared__ uint64_t best[kTopMax];
  __shared__ float red[kWaves];
  const long r = blockIdx.x;
  const Work w = work_of(p.workspace, p.in.rows, segs);
  const RowStats st = join_stats(w.stats + r * segs, segs, inv_t * kLog2e, red);
  if constexpr (DISTILL) {
    finish_distill<T>(p, r, st, inv_t, sh);
  } else {
    if (p.k > 0) join_top(w.keys + r * segs * p.k, segs, p.k, sh, best);
    finish_logprobs<T>(p, r, st, best, inv_t);
  }
}

// ------------------------------------------------------------------ backward kernels
// A workgroup to a segment, as in the forward pass: one read and one write. A row whose gradient is 0 is not read.
//
// p = e^(z - lse) is off by what rounding lse lost: with an |lse| below kFar at most 2^-16 of it, but with larger ones (logits far
// from 0, small temperatures) without bound, by any factor from some 2^23 on. Such a row is one workgroup's: it reads the row for
// its maximum and sum, from which p is taken as exactly as in the forward pass, and then goes through it in short segments (they
// need no more registers than the ordinary row's). One workgroup, as the gradients may take the logits' place. Half as much
// memory traffic again: 4096 rows of 32768 in fp32 283 us instead of 191; one row of 131072, with the other CUs idle, 45 instead of 8.2.
constexpr float kFar = 512.0f;
// Of such a row whose largest logit is this low nothing is left but masked columns (-inf or the type's lowest value): its p are
// taken as 0.
constexpr float kMasked = -0x1p100f;

// How ln p comes in base 2, of a logit x.
struct FromLse {
  float inv_t, lse;
  __device__ __forceinline__ float operator()(float x) const { return fmaf(x, inv_t, -lse) * kLog2e; }
};
struct FromMax {
  float m, c, log2_s;
  __device__ __forceinline__ float operator()(float x) const { return fmaf(x - m, c, -log2_s); }
};

__device__ __forceinline__ bool is_far(float lse) { return fabsf(lse) >= kFar; }  // not for NaN, whose gradients are NaN

// Of a whole row, by all threads of a workgroup; each thread sums over its own largest value so far.
constexpr int kFarPer = 16;  // values to a thread
template <typename T>
__device__ __forceinline__ FromMax read_row(const T *row, long cols, float c, float *red) {
  float m = -INFINITY, s = 0.0f;
  for (long col0 = 0; col0 < cols; col0 += kThreads * kFarPer) {
    Segment<T, kFarPer> x;
    x.load(row + col0, (int)min(cols - col0, (long)kThreads * kFarPer));
    const float n = fmaxf(m, x.max_value());
    if (n == -INFINITY) continue;
    s *= exp2_of((m - n) * c);
#pragma unroll
    for (int e = 0; e < kFarPer; ++e) s += exp2_of((x[e] - n) * c);
    m = n;
  }
  const float n = block_max(m, red);
  s = block_sum(m == -INFINITY ? 0.0f : s * exp2_of((m - n) * c), red);
  return {n, c, log2f(s)};
}

// f(a segment's first column, its values to a thread, ln p) for what is this workgroup's: segment seg of row r with p from its lse,
// or where that is far from 0 all of the row for one segment's workgroup (not always the first: workgroups next to each
// other run on different XCDs, whose number segs may be a multiple of). The last argument of f is true for a row of masked columns.
template <typename T, int E, typename F>
__device__ __forceinline__ void for_segments(const LogitsDesc &in, long r, int seg, int segs, float inv_t, float lse, bool far,
                                             float *red, F f) {
  if (!far) {
    f((long)seg * kThreads * E, std::integral_constant<int, E>{}, FromLse{inv_t, lse}, false);
  } else if (seg == (r + r / 8) % segs) {
    const FromMax p = read_row(static_cast<const T *>(in.x) + r * in.ld, in.cols, inv_t * kLog2e, red);
    const bool masked = p.m <= kMasked;
#pragma unroll 1
    for (long col0 = 0; col0 < in.cols; col0 += kThreads * kFarPer) f(col0, std::integral_constant<int, kFarPer>{}, p, masked);
  }
}

template <typename T, int E>
__global__ void __launch_bounds__(kThreads) logprobs_backward_kernel(LogprobsGradDesc p, float inv_t, int segs) {
  __shared__ float red[kWaves];
  const long r = blockIdx.x / segs;
  const T *row = static_cast<const T *>(p.in.x) + r * p.in.ld;
  const long t = p.targets ? p.targets[r] : -1;
  const float lse = p.lse[r], gh = p.grad_entropy ? p.grad_entropy[r] : 0.0f, h = p.grad_entropy ? p.entropy[r] : 0.0f;
  float gl = t >= 0 ? p.grad_logprob[r] : 0.0f;
  if (t >= p.in.cols) gl = NAN;
  const bool zero = gl == 0.0f && gh == 0.0f;
  const bool far = !zero && is_far(lse);
  for_segments<T, E>(p.in, r, blockIdx.x % segs, segs, inv_t, lse, far, red, [&](long col0, auto per, auto log2_p, bool masked) {
    constexpr int N = decltype(per)::value;
    const int left = (int)min(p.in.cols - col0, (long)kThreads * N);
    Segment<T, N> x;
    if (zero || (masked && t < p.in.cols)) {
#pragma unroll
      for (int i = 0; i < N / kVec<T>; ++i) x.v[i] = 0;
    } else {
      x.load(row + col0, left);
      const int at = t >= col0 && t < col0 + left ? (int)(t - col0) : -1;
      // In base 2: ln p = d ln 2. With the entropy's gradient as a and b: -p (gl + gh (ln p + h)) / T = p (a + b d).
      const float a = -(gl + gh * h) * inv_t, b = -gh * kLn2 * inv_t;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float d = log2_p(x[e]);
        float v = exp2_of(d) * fmaf(fmaxf(d, kFloor), b, a);  // 0 where p is 0 and d is -inf
        if (position<T>(e) == at) v += gl * inv_t;
        x.v[e / kVec<T>][e % kVec<T>] = (T)v;
      }
    }
    x.store(static_cast<T *>(p.grad) + r * p.ldg + col0, left);
  });
}

template <typename T, int E>
__global__ void __launch_bounds__(kThreads) distill_backward_kernel(DistillDesc p, float inv_t, int segs) {
  __shared__ Teacher sh;
  const long r = blockIdx.x / segs;
  const T *row = static_cast<const T *>(p.in.x) + r * p.in.ld;
  const float gt = p.grad_loss[r] * p.in.temperature, lse = p.lse_in[r];
  const Entry entry = load_entry(p, r);  // before the segment: loads arrive in order
  bool known = false, some = false;
  const bool far = gt != 0.0f && is_far(lse);
  for_segments<T, E>(p.in, r, blockIdx.x % segs, segs, inv_t, lse, far, sh.red, [&](long col0, auto per, auto log2_p, bool masked) {
    constexpr int N = decltype(per)::value;
    const int left = (int)min(p.in.cols - col0, (long)kThreads * N);
    T *out = static_cast<T *>(p.grad) + r * p.ldg + col0;
    Segment<T, N> x;
    if (gt != 0.0f) x.load(row + col0, left);
    if (!known) some = teacher_row(p, entry, inv_t, sh), known = true;
    const bool none = !some || gt == 0.0f;
    const float bad = some && sh.w[0] != sh.w[0] ? NAN : 0.0f;
    auto q = [&](float v) { return masked ? 0.0f : exp2_of(log2_p(v)); };
    // The entries of this segment are put right once the segment is written; their logits are read before (grad may be
    // the logits). An id may occur more than once: all of its occurrences write the same value.
    const int i = threadIdx.x;
    const long at = some && i < p.k ? sh.at[i] - col0 : -1;
    const bool mine = !none && at >= 0 && at < left;
    float fix = 0.0f;
    if (mine) {
      float sum = 0.0f;
#pragma unroll 8
      for (int j = 0; j < p.k; ++j) sum += sh.at[j] == sh.at[i] ? sh.w[j] : 0.0f;
      fix = gt * (q((float)row[col0 + at]) - sum + bad);
    }
    const bool any = __syncthreads_or(mine);
#pragma unroll
    for (int e = 0; e < N; ++e) x.v[e / kVec<T>][e % kVec<T>] = none ? (T)0.0f : (T)(gt * (q(x[e]) + bad));
    x.store(out, left);
    if (any) {
      __syncthreads();
      if (mine) out[at] = (T)fix;
    }
  });
}

// ------------------------------------------------------------------ host
int check_logits(const char *what, const LogitsDesc &d, CError *err) {
  size_t n;
  if (d.dtype != GN_F32 && d.dtype != GN_F16) return set_error(err, -1, "%s: unsupported dtype %d", what, d.dtype);
  if (d.rows < 0 || d.cols < 1 || d.cols > INT_MAX)
    return set_error(err, -1, "%s: invalid size %ld x %ld", what, d.rows, d.cols);
  // The kernels multiply by c = log2(e) / T, and 0 times an infinite one would be NaN.
  if (!(d.temperature > 0.0f) || !(1.0f / d.temperature > 0.0f) || !(1.0f / d.temperature * kLog2e < INFINITY))
    return set_error(err, -1, "%s: a temperature above 0 and finite, with a finite log2(e) / temperature, is needed", what);
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
// 131072, 20 alternatives: 16 workgroups of 8192 take 8.4 us and their join 7.4, 64 of 2048 6.2 and 7.1). Calls with 8 against 32, us
// (forward, with 20 alternatives, gradient; logits in the Infinity Cache): 1 x 131072 fp32 5.5 / 6.0, 12.6 / 15.7, 2.3 / 3.4; 16 x 131072
// 6.5 / 6.5, 14.4 / 16.2, 4.0 / 4.6; 32 x 131072, at the border, 7.5 / 7.1, 18.0 / 16.9, 5.4 / 6.8; 64 x 50257 fp16 7.3 / 7.5,
// 16.6 / 16.2, 4.6 / 5.6; 512 x 4096 fp32 6.9 / 4.6, 12.6 / 9.1, 4.0 / 5.5. Below the border rows of one segment of 8192 lose their join
// with 32 (256 x 8192 6.6 / 3.8, 12.8 / 8.9, 4.0 / 4.6): forward and gradient share the rule all the same.
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
