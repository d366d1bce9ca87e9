// adjust.hip — logits before sampling: penalties for the tokens so far, biases, masks; and the gradient of the logits.
//
// A workgroup takes a segment of a row. It counts the row's tokens that fall into the segment in LDS (whole numbers: the order
// in which they are added changes nothing), then goes once over the segment's logits, which were asked for before, and
// looks each one's count up. In place and without a mask only the counted tokens change: each is put right by one thread, whoever
// first sets a bit beside its count, and nothing else is read or written.
// What bounds them: with many rows memory (4096 x 32768 in fp32, out of place, 182 us, 5.9 TB/s; the gradient, from another tensor than its
// own, 216), with few the latencies of the tokens, of counting them and of what is looked up (1 x 131072 3.1 us, 64 x 50257 in fp16
// 5.2, with 2048 tokens and 64 biases to a row and a mask 7.9). In place without a mask, where the tokens and what they name is all that a call
// has to read, it is that every segment's workgroup reads all of its row's tokens: 256 x 131072 in fp16 with 1000 of them 25 us, several
// times what the bytes would take.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "adjust.h"
#include "int8_round.h"

namespace gn {
namespace {

constexpr int kMaxBiases = 1024;
constexpr int kPer = 8;  // logits to a thread

template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

// A thread's vectors of a segment: vector i holds the segment's values at place<T>(i) and after it.
template <typename T, int NT>
__device__ __forceinline__ int place(int i) {
  return (i * NT + (int)threadIdx.x) * kVec<T>;
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

// The mask's word with the bits of the kVec columns from `col` on (a multiple of kVec); ones without a mask. Its bits are not touched
// here, which would be a wait for it.
__device__ __forceinline__ uint32_t mask_word(const uint32_t *mask, long col, long cols) {
  return mask ? mask[min(col, cols - 1) >> 5] : ~0u;
}

// A vector's masked values.
template <typename T>
__device__ __forceinline__ void apply_mask(Vector<T> &v, uint32_t word, long col, T masked) {
  const uint32_t bits = word >> (col & 31);
  constexpr uint32_t ALL = (1u << kVec<T>) - 1;
  if ((bits & ALL) == ALL) return;
#pragma unroll
  for (int j = 0; j < kVec<T>; ++j)
    if (!((bits >> j) & 1)) v.v[j] = masked;
}

// A thread's value number j of all of its vectors', and that value replaced, without memory: a choice among its registers.
template <typename T, int VECS>
__device__ __forceinline__ T value_of(const Vector<T> (&v)[VECS], int j) {
  constexpr int PER = 4 / (int)sizeof(T);
  uint32_t w = 0;
#pragma unroll
  for (int k = 0; k < 4 * VECS; ++k) {
    const u32x4_t four = __builtin_bit_cast(u32x4_t, v[k / 4].v);
    w |= four[k % 4] & (j / PER == k ? ~0u : 0u);
  }
  if constexpr (PER == 1)
    return __uint_as_float(w);
  else
    return __builtin_bit_cast(T, (uint16_t)(w >> (16 * (j % PER))));
}
template <typename T, int VECS>
__device__ __forceinline__ void replace(Vector<T> (&v)[VECS], int j, T y) {
  constexpr int PER = 4 / (int)sizeof(T);
  uint32_t bits, mask;
  if constexpr (PER == 1)
    bits = __float_as_uint(y), mask = ~0u;
  else
    bits = (uint32_t)__builtin_bit_cast(uint16_t, y) << (16 * (j % PER)), mask = 0xffffu << (16 * (j % PER));
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    u32x4_t w = __builtin_bit_cast(u32x4_t, v[i].v);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t m = j / PER == 4 * i + k ? mask : 0u;
      w[k] = (w[k] & ~m) | (bits & m);
    }
    v[i].v = __builtin_bit_cast(decltype(v[i].v), w);
  }
}

// This thread's share of a row's tokens, kTokens at a time, token u being the row's number i + u NT (-1 past its end): their loads
// are in flight together, those of the first ones from the kernel's start.
constexpr int kTokens = 4;
template <int NT>
struct Tokens {
  const int64_t *ids;
  int n;  // below 2^29: a token's place in bytes fits 32 bits
  int64_t id[kTokens];
  __device__ __forceinline__ Tokens(const int64_t *row, long h) : ids(row), n((int)h) { load(threadIdx.x); }
  __device__ __forceinline__ void load(int i0) {
#pragma unroll
    for (int u = 0; u < kTokens; ++u) {
      const int i = i0 + u * NT;
      id[u] = i < n ? *reinterpret_cast<const int64_t *>(reinterpret_cast<const char *>(ids) + 8u * (unsigned)i) : -1;
    }
  }
  // f(tokens, i) for all of them, the first of which are there.
  template <typename F>
  __device__ __forceinline__ void each(F f) {
    for (int i0 = threadIdx.x; i0 < n;) {
      f(id, i0);
      i0 += kTokens * NT;
      if (i0 < n) load(i0);
    }
  }
  __device__ __forceinline__ void again() {
    if (n > kTokens * NT) load(threadIdx.x);
  }
};

// A token's column in the segment of `left` columns from col0 on, if it is below `left`.
__device__ __forceinline__ unsigned place_of(int64_t id, long col0) {
  const unsigned at = (unsigned)id - (unsigned)col0;
  return (uint64_t)id >> 32 ? ~0u : at;
}

// What a column's cell of the counts says: bit 31 in the prompt, bit 30 there is a bias, bit 29 it has been put right, below them how
// often in the answer. Until its biases are added up, bit 29 says that it has several.
constexpr uint32_t kPrompt = 1u << 31, kBiased = 1u << 30, kDone = 1u << 29, kSeveral = kDone, kCount = kDone - 1;

// A row's penalties.
struct Penalties {
  float rho, freq, pres;
  // y of a counted token, whose biases' sum is `bias` where it has some. No product is left open to be taken with the sum after it.
  __device__ __forceinline__ float operator()(float y, uint32_t cell, float bias) const {
    const uint32_t n = cell & kCount;
    if (n != 0 || (cell & kPrompt)) y = y > 0.0f ? y / rho : as_fp32(y * rho);
    if (n != 0) y = (y - as_fp32(freq * (float)n)) - pres;
    if (cell & kBiased) y = as_fp32(y) + bias;
    return as_fp32(y);
  }
};

// PATCH: in place and without a mask.
template <typename T, int NT, bool BIASES, bool PATCH>
__global__ void __launch_bounds__(NT) adjust_kernel(AdjustDesc p, int segs) {
  constexpr int SEG = NT * kPer, VECS = kPer / kVec<T>;
  __shared__ __attribute__((aligned(16))) uint32_t cells[SEG];
  __shared__ float sums[BIASES ? SEG : 1];  // of a token's biases, where its cell says that there are some
  __shared__ int again, hit;  // a token has several biases; there is one in the segment
  const long r = blockIdx.x / segs;
  const long col0 = (long)(blockIdx.x % segs) * SEG;
  const int left = (int)min(p.cols - col0, (long)SEG);
  const T *x = static_cast<const T *>(p.x) + r * p.ld + col0;
  T *out = static_cast<T *>(p.out) + r * p.ldo + col0;
  const int64_t *history = p.history + r * p.h, *bias_ids = p.bias_ids + r * p.biases;
  const float *bias = p.bias + r * p.biases;
  // All that has to come from memory is asked for before anything is waited for.
  const Penalties penalty{p.repetition ? p.repetition[r] : 1.0f, p.frequency ? p.frequency[r] : 0.0f, p.presence ? p.presence[r] : 0.0f};
  const int prompt = p.prompt ? (int)min((int64_t)p.h, max((int64_t)0, p.prompt[r])) : 0;
  Tokens<NT> tokens(history, p.h);
  int64_t bias_id = -1;  // the row's bias threadIdx.x
  float bias_value = 0.0f;
  if (BIASES && (int)threadIdx.x < p.biases) bias_id = bias_ids[threadIdx.x], bias_value = bias[threadIdx.x];
  Vector<T> v[PATCH ? 1 : VECS];
  uint32_t words[PATCH ? 1 : VECS];
  if constexpr (!PATCH) {
    const uint32_t *mask = p.mask ? p.mask + r * p.ldmask : nullptr;
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int at = place<T, NT>(i);
      words[i] = mask_word(mask, col0 + at, p.cols);
      v[i].load(x + at, left - at);
    }
  }
#pragma unroll
  for (int i = 0; i < kPer / 4; ++i) reinterpret_cast<u32x4_t *>(cells)[i * NT + threadIdx.x] = u32x4_t{0, 0, 0, 0};
  if (threadIdx.x == 0) again = hit = 0;
  __syncthreads();
  bool any = false;
  tokens.each([&](const int64_t (&id)[kTokens], int i0) {
#pragma unroll
    for (int u = 0; u < kTokens; ++u) {
      const unsigned at = place_of(id[u], col0);
      if (at < (unsigned)left) {
        any = true;
        if (i0 + u * NT < prompt)
          atomicOr(&cells[at], kPrompt);
        else
          atomicAdd(&cells[at], 1u);
      }
    }
  });
  if constexpr (BIASES) {
    for (int i = threadIdx.x; i < p.biases; i += NT) {
      const unsigned at = place_of(i < NT ? bias_id : bias_ids[i], col0);
      if (at < (unsigned)left) {
        any = true;
        if (atomicOr(&cells[at], kBiased) & kBiased) {
          atomicOr(&cells[at], kSeveral);
          again = 1;
        } else {
          sums[at] = i < NT ? bias_value : bias[i];
        }
      }
    }
  }
  if (any) hit = 1;
  __syncthreads();
  const bool touched = hit;
  // The biases of a token that has several are added up anew by the first wave, one after the other. A sum goes from lane to lane through
  // LDS, which keeps a wave's order; so has the compiler to.
  if constexpr (BIASES) {
    if (again) {
      if (threadIdx.x < 64) {
        auto several = [&](int i) {
          const unsigned at = i >= p.biases ? ~0u : place_of(i < 64 ? bias_id : bias_ids[i], col0);
          return at < (unsigned)left && (cells[at] & kSeveral) ? (int)at : -1;
        };
        for (int i = threadIdx.x; i < p.biases; i += 64) {
          const int at = several(i);
          if (at >= 0) sums[at] = 0.0f;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        for (int i0 = 0; i0 < p.biases; i0 += 64) {
          const int i = i0 + threadIdx.x, at = several(i);
          const float b = at < 0 ? 0.0f : i < 64 ? bias_value : bias[i];
          for (uint64_t here = __ballot(at >= 0); here != 0; here &= here - 1) {
            if ((int)threadIdx.x == __ffsll((unsigned long long)here) - 1) sums[at] += b;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          }
        }
        for (int i = threadIdx.x; PATCH && i < p.biases; i += 64) {
          const int at = several(i);
          if (at >= 0) atomicAnd(&cells[at], ~kSeveral);
        }
      }
      __syncthreads();
    }
  }
  if constexpr (PATCH) {
    auto patch = [&](unsigned at) {
      if (at >= (unsigned)left) return;
      const uint32_t cell = atomicOr(&cells[at], kDone);
      if (!(cell & kDone)) out[at] = (T)penalty((float)out[at], cell, BIASES ? sums[at] : 0.0f);
    };
    if (touched) {
      tokens.again();
      tokens.each([&](const int64_t (&id)[kTokens], int) {
#pragma unroll
        for (int u = 0; u < kTokens; ++u) patch(place_of(id[u], col0));
      });
      if constexpr (BIASES)
        for (int i = threadIdx.x; i < p.biases; i += NT) patch(place_of(bias_ids[i], col0));
    }
  } else {
    if (touched) {
      // The lanes' counted values one after the other: few rounds for a wave, as each lane has few. (All eight values in turn, those of any
      // lane computed: 64 x 50257 with 2048 tokens 8.5 us instead of 7.9, 1 x 131072 3.2 / 3.1; only where the tokens are as many as half of the
      // columns, 2048 x 8192 with 4096 of them, less: 31.7 / 34.3.)
      uint32_t counted = 0;
#pragma unroll
      for (int j0 = 0; j0 < kPer; j0 += 4) {
        const u32x4_t four = *reinterpret_cast<const u32x4_t *>(cells + place<T, NT>(j0 / kVec<T>) + j0 % kVec<T>);
#pragma unroll
        for (int e = 0; e < 4; ++e) counted |= four[e] != 0 ? 1u << (j0 + e) : 0u;
      }
      for (; counted != 0; counted &= counted - 1) {
        const int j = __ffs(counted) - 1, at = place<T, NT>(j / kVec<T>) + j % kVec<T>;
        replace(v, j, (T)penalty((float)value_of(v, j), cells[at], BIASES ? sums[at] : 0.0f));
      }
    }
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int at = place<T, NT>(i);
      if (at >= left) break;
      apply_mask(v[i], words[i], col0 + at, (T)-INFINITY);
      v[i].store(out + at, left - at);
    }
  }
}

// The gradient of a logit is that of the adjusted one times 1, or rho or 1 / rho by the logit's sign where the token is among
// those so far, or 0 where it is masked. PATCH: in the gradient's place, without a mask.
template <typename T, int NT, bool PATCH>
__global__ void __launch_bounds__(NT) adjust_backward_kernel(AdjustGradDesc p, int segs) {
  constexpr int SEG = NT * kPer, VECS = kPer / kVec<T>;
  __shared__ uint32_t seen[SEG / 32], positive[SEG / 32];  // bits: a token so far, and whether its logit is above 0
  __shared__ int hit;                                      // there is one in the segment
  const long r = blockIdx.x / segs;
  const long col0 = (long)(blockIdx.x % segs) * SEG;
  const int left = (int)min(p.cols - col0, (long)SEG);
  const T *x = static_cast<const T *>(p.x) + r * p.ld + col0, *g = static_cast<const T *>(p.grad_out) + r * p.ldg + col0;
  T *out = static_cast<T *>(p.grad) + r * p.ldo + col0;
  const bool counts = p.repetition && p.h > 0;
  const float rho = p.repetition ? p.repetition[r] : 1.0f;
  auto factored = [&](T d, bool above) { return (T)as_fp32(above ? (float)d / rho : (float)d * rho); };
  Tokens<NT> tokens(p.history + r * p.h, counts ? p.h : 0);
  Vector<T> v[PATCH ? 1 : VECS];
  uint32_t words[PATCH ? 1 : VECS];
  if constexpr (!PATCH) {
    const uint32_t *mask = p.mask ? p.mask + r * p.ldmask : nullptr;
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int at = place<T, NT>(i);
      words[i] = mask_word(mask, col0 + at, p.cols);
      v[i].load(g + at, left - at);
    }
  }
  bool any = false;
  if (counts) {
    if (threadIdx.x == 0) hit = 0;
    for (int i = threadIdx.x; i < SEG / 32; i += NT) seen[i] = positive[i] = 0;
    __syncthreads();
    // Whoever sets a token's bit first asks for its logit. They are read before anything is written: the
    // gradient may take their place.
    tokens.each([&](const int64_t (&id)[kTokens], int) {
      int at[kTokens];
      float z[kTokens];
#pragma unroll
      for (int u = 0; u < kTokens; ++u) {
        const unsigned a = place_of(id[u], col0);
        at[u] = -1;
        if (a < (unsigned)left && !(atomicOr(&seen[a >> 5], 1u << (a & 31)) & (1u << (a & 31)))) at[u] = (int)a, any = true;
      }
#pragma unroll
      for (int u = 0; u < kTokens; ++u) z[u] = at[u] >= 0 ? (float)x[at[u]] : 0.0f;
#pragma unroll
      for (int u = 0; u < kTokens; ++u) {
        if (PATCH) {
          if (at[u] >= 0) out[at[u]] = factored(out[at[u]], z[u] > 0.0f);
        } else if (z[u] > 0.0f) {
          atomicOr(&positive[at[u] >> 5], 1u << (at[u] & 31));
        }
      }
    });
  }
  if constexpr (!PATCH) {
    if (any) hit = 1;
    if (counts) __syncthreads();
    const bool touched = counts && hit;
    if (touched) {
      uint32_t here = 0, above = 0;
#pragma unroll
      for (int i = 0; i < VECS; ++i) {
        const int at = place<T, NT>(i);
        here |= (seen[at >> 5] >> (at & 31) & ((1u << kVec<T>) - 1)) << (i * kVec<T>);
        above |= (positive[at >> 5] >> (at & 31) & ((1u << kVec<T>) - 1)) << (i * kVec<T>);
      }
      for (; here != 0; here &= here - 1) {
        const int j = __ffs(here) - 1;
        replace(v, j, factored(value_of(v, j), (above >> j) & 1));
      }
    }
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int at = place<T, NT>(i);
      if (at >= left) break;
      apply_mask(v[i], words[i], col0 + at, (T)0.0f);
      v[i].store(out + at, left - at);
    }
  }
}

// ------------------------------------------------------------------ host
// Threads to a workgroup: 256, 2048 logits, or 1024 where the row's tokens, all of which every workgroup reads, are many. Kernels with
// 256 and with 1024, us (forward, gradient): 1 x 131072 fp32, 300 tokens 3.1 / 3.7, 3.2 / 3.7; 64 x 50257 fp16, 100 tokens 5.2 / 5.4,
// 5.2 / 5.3, 1000 tokens 6.0 / 6.2, 6.9 / 6.2, 2048 tokens 7.9 / 7.0, 9.3 / 7.5; 256 x 131072 fp16, 1000 tokens 27.3 / 31.6, 31.2 / 31.2, 1500 tokens
// 31.5 / 31.9, 38.9 / 33.1; 16 x 131072, 4000 tokens 6.0 / 4.7, 8.8 / 5.5; 2048 x 8192, 4096 tokens 51 / 33, 65 / 42; 1 x 131072, 100000 tokens
// 43 / 18, 70 / 28; 4096 x 32768 fp32, 512 tokens 185 / 191, 219 / 220. (32 logits to each of 256 threads: 229 us where 8 took 207.)
// In place without a mask the kernels that touch only the tokens' columns are taken (PATCH). They and those that pass over the row, both in place,
// us (forward, gradient): 1 x 131072 fp32, 300 tokens 2.8 / 3.1, 2.5 / 3.2; 64 x 50257 fp16, 100 tokens 3.8 / 5.4, 3.4 / 5.3, 1000 tokens
// 5.4 / 6.0, 5.9 / 6.8, 2048 tokens 5.6 / 7.0, 5.6 / 7.7; 256 x 131072 fp16, 1000 tokens 25 / 28, 25 / 32; 16 x 131072, 4000 tokens 4.4 / 4.6, 4.9 / 5.5;
// 2048 x 8192, 1500 tokens 18 / 23, 23 / 27; 4096 x 32768 fp32, 512 tokens 90 / 188, 115 / 223. They are the slower ones for long histories, 2048 x
// 8192, 4096 tokens 36 / 30, 49 / 40; 1 x 131072, 20000 tokens 11.0 / 6.8, 9.6 / 9.1, 100000 tokens 40 / 18, 33 / 29: no border is drawn there.
constexpr long kManyTokens = 1024;
struct Split {
  int nt, segs;
};
Split split_of(long cols, long h) {
  const int nt = h < kManyTokens ? 256 : 1024;
  return {nt, (int)((cols + nt * kPer - 1) / (nt * kPer))};
}

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
  const Split sp = split_of(cols, h);
  if (rows > ((1L << 32) / sp.nt - 1) / sp.segs) return set_error(err, -1, "%s: %ld x %ld is too large", what, rows, cols);  // threads
  // Counts stay below the bits that stand beside them.
  if (h < 0 || h >= (long)kDone || !matrix_bytes(rows, h, 8, &n)) return set_error(err, -1, "%s: history of %ld tokens", what, h);
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

// f(type, threads, biases, patch) with all of them as types.
template <typename F>
void with_kind(int dtype, int nt, bool biases, bool patch, F f) {
  auto flag = [](bool v, auto g) {
    if (v)
      g(std::true_type{});
    else
      g(std::false_type{});
  };
  flag(dtype == GN_F16, [&](auto half) {
    flag(nt == 256, [&](auto few) {
      flag(biases, [&](auto b) {
        flag(patch, [&](auto c) {
          f(std::conditional_t<decltype(half)::value, _Float16, float>{}, std::integral_constant<int, decltype(few)::value ? 256 : 1024>{}, b, c);
        });
      });
    });
  });
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
  if ((uintptr_t)d.prompt % 8 || (uintptr_t)d.repetition % 4 || (uintptr_t)d.frequency % 4 || (uintptr_t)d.presence % 4)
    return set_error(err, -1, "%s: prompt lengths or penalties not aligned to their type", what);
  if (d.biases > 0 && (!d.bias_ids || !d.bias)) return set_error(err, -1, "%s: NULL biases", what);
  if ((uintptr_t)d.bias_ids % 8 || (uintptr_t)d.bias % 4) return set_error(err, -1, "%s: biases not aligned to their type", what);
  return 0;
}

int launch_adjust(const AdjustDesc &d, hipStream_t s, CError *err) {
  if (d.rows == 0) return 0;
  const Split sp = split_of(d.cols, d.h);
  with_kind(d.dtype, sp.nt, d.biases > 0, d.out == d.x && !d.mask, [&](auto type, auto nt, auto biases, auto patch) {
    hipLaunchKernelGGL((adjust_kernel<decltype(type), decltype(nt)::value, decltype(biases)::value, decltype(patch)::value>),
                       dim3((unsigned)(d.rows * sp.segs)), dim3(sp.nt), 0, s, d, sp.segs);
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
  const Split sp = split_of(d.cols, d.h);
  with_kind(d.dtype, sp.nt, false, d.grad == d.grad_out && !d.mask, [&](auto type, auto nt, auto, auto patch) {
    hipLaunchKernelGGL((adjust_backward_kernel<decltype(type), decltype(nt)::value, decltype(patch)::value>),
                       dim3((unsigned)(d.rows * sp.segs)), dim3(sp.nt), 0, s, d, sp.segs);
  });
  return launched("adjust logits backward launch", err);
}

}  // namespace gn
