// int8_gemm.hip — products of 8-bit integers, C = act(alpha (sum_k A B) b_scale a_scale + beta C + bias).
//
// The sums are exact in 32 bits (K below 2^17). A sum becomes fp32 and is multiplied by its column's scale and then by
// its row's, each rounded once.
#include <algorithm>
#include <climits>

#include "gemm_tile.h"
#include "int8.h"

namespace gn {
namespace {

// 256 rows stay below 2^31 bytes: 32-bit offsets within a tile.
constexpr long kMaxLd = 1L << 22, kMaxRows = 1L << 25;

struct Int8Params : GemmParams {
  const float *as, *bs;  // scales; NULL: 1
};

// c + A B^T of 16 x 64 integers each: lane (r, g) = (lane % 16, lane / 16) has 16 of row r's k, the same ones on both sides.
__device__ __forceinline__ i32x4_t mfma_i8(i32x4_t a, i32x4_t b, i32x4_t c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

// The first `n` bytes of v, zeros after them.
__device__ __forceinline__ i32x4_t first_bytes(i32x4_t v, int n) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int left = n - 4 * i;
    v[i] = left >= 4 ? v[i] : left <= 0 ? 0 : v[i] & ((1 << (8 * left)) - 1);
  }
  return v;
}

__device__ __forceinline__ float finish(const Int8Params &p, float v, long m, long n) {
  v *= p.alpha;
  if (p.beta != 0.0f) v += p.beta * p.C[m * p.ldc + n];
  if (p.bias) v += p.bias[n];
  return apply_act(p.act, v, p.act_alpha);
}

// K == 0: act(beta C + bias).
__global__ void __launch_bounds__(256) i8_k0_kernel(Int8Params p) {
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < p.M * p.N; i += (long)gridDim.x * 256)
    p.C[i / p.N * p.ldc + i % p.N] = finish(p, 0.0f, i / p.N, i % p.N);
}

// ------------------------------------------------------------------ few rows
// A workgroup takes all rows (MF blocks of 16) and 16 NF columns; its KW waves take steps of 128 k in turn, each with D
// steps of A and B in registers, and their sums meet in LDS. Rows and columns past the matrix are the last ones again, not stored.
template <int MF, int NF, int KW, int D>
__global__ void __launch_bounds__(KW * 64) i8_rows_kernel(Int8Params p) {
  __shared__ i32x4_t part[KW][MF * NF][64];
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const long n0 = (long)blockIdx.x * 16 * NF, m0 = (long)blockIdx.y * 16 * MF;
  const int8_t *ap[MF], *bp[NF];
#pragma unroll
  for (int i = 0; i < MF; ++i) ap[i] = static_cast<const int8_t *>(p.A) + min(m0 + 16 * i + r, p.M - 1) * p.lda + 16 * g;
#pragma unroll
  for (int j = 0; j < NF; ++j) bp[j] = static_cast<const int8_t *>(p.B) + min(n0 + 16 * j + r, p.N - 1) * p.ldb + 16 * g;
  i32x4_t acc[MF][NF];
#pragma unroll
  for (int i = 0; i < MF; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) acc[i][j] = i32x4_t{0, 0, 0, 0};

  i32x4_t a[D][2][MF], b[D][2][NF];
  auto load = [&](int d, long k) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int j = 0; j < NF; ++j) b[d][h][j] = *reinterpret_cast<const i32x4_t *>(bp[j] + k + 64 * h);
#pragma unroll
      for (int i = 0; i < MF; ++i) a[d][h][i] = *reinterpret_cast<const i32x4_t *>(ap[i] + k + 64 * h);
    }
  };
  auto multiply = [&](int d) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int j = 0; j < NF; ++j) acc[i][j] = mfma_i8(a[d][h][i], b[d][h][j], acc[i][j]);
  };
  const int full = (int)(p.K / 128);  // whole steps; this wave has steps wave, wave + KW, ...
  const int mine = wave < full ? (full - wave + KW - 1) / KW : 0;
  const long k0 = 128L * wave;
#pragma unroll
  for (int d = 0; d < D; ++d)
    if (d < mine) load(d, k0 + 128L * KW * d);
  for (int t = 0; t < mine; t += D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      if (t + d >= mine) break;
      multiply(d);
      if (t + d + D < mine) load(d, k0 + 128L * KW * (t + d + D));
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  // The rest of K: chunks of 16 that begin inside it (their other bytes belong to the rows too), A's bytes past K as zeros.
  if (p.K % 128 != 0 && wave == full % KW) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const long k = 128L * full + 64 * h;
      const int left = (int)(p.K - k) - 16 * g;  // of this lane's chunk
#pragma unroll
      for (int j = 0; j < NF; ++j) b[0][h][j] = left > 0 ? *reinterpret_cast<const i32x4_t *>(bp[j] + k) : i32x4_t{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < MF; ++i)
        a[0][h][i] = left > 0 ? first_bytes(*reinterpret_cast<const i32x4_t *>(ap[i] + k), left) : i32x4_t{0, 0, 0, 0};
    }
    multiply(0);
  }
#pragma unroll
  for (int i = 0; i < MF; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) part[wave][i * NF + j][lane] = acc[i][j];
  __syncthreads();
  for (int f = wave; f < MF * NF; f += KW) {
    i32x4_t v = part[0][f][lane];
#pragma unroll
    for (int w = 1; w < KW; ++w) v += part[w][f][lane];
    const long n = n0 + 16 * (f % NF) + r;
    if (n >= p.N) continue;
    const float bs = p.bs ? p.bs[n] : 1.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const long m = m0 + 16 * (f / NF) + 4 * g + e;
      if (m < p.M) p.C[m * p.ldc + n] = finish(p, (float)v[e] * bs * (p.as ? p.as[m] : 1.0f), m, n);
    }
  }
}

// ------------------------------------------------------------------ many rows
// WM x WN waves, each FM x FN blocks of 16 x 16. K goes in stages of 128 bytes to a row, copied straight to LDS by dma16 in chunks
// of 8 rows (ring_plan.h's places: a wave's copies are whole 128-byte lines, its fragment reads fall on distinct banks), NS stages
// in LDS. A stage is two steps of 64 k: while one is multiplied the next one's fragments are read, and before the
// second the next stage has landed (one wait and one barrier to a stage) and the copies of the one NS ahead start.
// Where K ends inside a chunk of 16 the wave that copied it clears A's bytes past K before that barrier.
template <int WM, int WN, int FM, int FN, int NS, int WPE>
__global__ void __launch_bounds__(WM * WN * 64) __attribute__((amdgpu_waves_per_eu(WPE, WPE)))
i8_tile_kernel(Int8Params p) {
  constexpr int NW = WM * WN, NT = NW * 64, BM = WM * FM * 16, BN = WN * FN * 16;
  constexpr int CA = BM / 8 / NW, CB = BN / 8 / NW, CPW = CA + CB;
  constexpr int STAGE = (BM + BN) * 128, EPI = WM * 16 * (BN + 4) * 4;
  static_assert(CA * NW * 8 == BM && CB * NW * 8 == BN && CA % 2 == 0 && CB % 2 == 0, "chunks");
  static_assert(EPI + (BM + BN) * 4 <= NS * STAGE && (NS - 1) * CPW < 64 && NS >= 2, "LDS");
  __shared__ __attribute__((aligned(1024))) char smem[NS * STAGE];

  int tm, tn;
  tile_coords(p, tm, tn);
  const long m0 = (long)tm * BM, n0 = (long)tn * BN;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wm = wave / WN, wn = wave % WN, r = lane & 15, g = lane >> 4;
  const int ns = (int)((p.K + 127) / 128);

  // The tile's scales: A's, then B's, thread by thread; in LDS once the stages are done with it.
  constexpr int SPT = (BM + BN + NT - 1) / NT;
  float scale[SPT];
#pragma unroll
  for (int i = 0; i < SPT; ++i) {
    const int at = threadIdx.x + i * NT;
    scale[i] = 1.0f;
    if (at < BM) {
      if (p.as && m0 + at < p.M) scale[i] = p.as[m0 + at];
    } else if (at < BM + BN) {
      if (p.bs && n0 + at - BM < p.N) scale[i] = p.bs[n0 + at - BM];
    }
  }

  const char *a0 = static_cast<const char *>(p.A) + m0 * p.lda, *b0 = static_cast<const char *>(p.B) + n0 * p.ldb;
  unsigned va[CA], vb[CB];
  // A copy's first k in the stage, for even i; for odd i the octet's upper bit is the other way round (row >> 1 is 4 more).
  const int ka = 16 * kc8_octet(8 * wave * CA + (lane >> 3), lane & 7), kb = 16 * kc8_octet(8 * wave * CB + (lane >> 3), lane & 7);
  auto k_of = [](int k, int i) { return k ^ (i & 1 ? 64 : 0); };
#pragma unroll
  for (int i = 0; i < CA; ++i) {
    const int row = 8 * (wave * CA + i) + (lane >> 3);
    va[i] = m0 + row < p.M ? (unsigned)(row * p.lda) + k_of(ka, i) : kOutOfRange;
  }
#pragma unroll
  for (int i = 0; i < CB; ++i) {
    const int row = 8 * (wave * CB + i) + (lane >> 3);
    vb[i] = n0 + row < p.N ? (unsigned)(row * p.ldb) + k_of(kb, i) : kOutOfRange;
  }
  const unsigned lds = lds_offset(smem);
  // Copies of a stage; chunks that begin at or past K read zeros.
  auto issue = [&](const char *base, const unsigned *v, int k, int count, int t, unsigned to) {
    const int left = (int)p.K - 128 * t;
    const BufRsrc d = make_rsrc(base + 128L * t);
    if (left >= 128) {
#pragma unroll
      for (int i = 0; i < count; ++i) dma16(d, v[i], __builtin_amdgcn_readfirstlane(to + i * 1024));
    } else {
#pragma unroll
      for (int i = 0; i < count; ++i) dma16(d, k_of(k, i) < left ? v[i] : kOutOfRange, __builtin_amdgcn_readfirstlane(to + i * 1024));
    }
  };
  auto issue_a = [&](int t, int slot) { issue(a0, va, ka, CA, t, lds + slot * STAGE + wave * CA * 1024); };
  auto issue_b = [&](int t, int slot) { issue(b0, vb, kb, CB, t, lds + slot * STAGE + BM * 128 + wave * CB * 1024); };
  // This wave's chunks of A of the last stage, once they have landed (all that is under way behind them reads zeros).
  auto clear_tail = [&](int slot) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const int left = (int)p.K - 128 * (ns - 1);
#pragma unroll
    for (int i = 0; i < CA; ++i) {
      const int n = left - k_of(ka, i);
      if (n > 0 && n < 16) {
        i32x4_t *c = reinterpret_cast<i32x4_t *>(smem + slot * STAGE + (wave * CA + i) * 1024 + lane * 16);
        *c = first_bytes(*c, n);
      }
    }
  };

  i32x4_t fa[2][FM], fb[2][FN];
  auto read_a = [&](int slot, int h, int i) {
    const int row = (wm * FM + i) * 16 + r;
    fa[h][i] = *reinterpret_cast<const i32x4_t *>(smem + slot * STAGE + (row >> 3) * 1024 + 16 * kc8_slot(row, 4 * h + g));
  };
  auto read_b = [&](int slot, int h, int j) {
    const int row = (wn * FN + j) * 16 + r;
    fb[h][j] = *reinterpret_cast<const i32x4_t *>(smem + slot * STAGE + BM * 128 + (row >> 3) * 1024 + 16 * kc8_slot(row, 4 * h + g));
  };
  auto read_part = [&](int slot, int h, int q, int parts) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
      if (i * parts / FM == q) read_a(slot, h, i);
#pragma unroll
    for (int j = 0; j < FN; ++j)
      if (j * parts / FN == q) read_b(slot, h, j);
  };
  i32x4_t acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = i32x4_t{0, 0, 0, 0};
  auto mfma_rows = [&](int h, int i0, int i1) {
#pragma unroll
    for (int i = i0; i < i1; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = mfma_i8(fa[h][i], fb[h][j], acc[i][j]);
  };

  const bool tail = p.K % 16 != 0;
#pragma unroll
  for (int t = 0; t < NS; ++t) {
    issue_a(t, t);
    issue_b(t, t);
  }
  __builtin_amdgcn_s_waitcnt(vmcnt_imm((NS - 1) * CPW));
  if (tail && ns == 1) clear_tail(0);
  __syncthreads();
  read_part(0, 0, 0, 1);
  int cur = 0;
  for (int t = 0; t < ns; ++t) {
    const int nxt = cur + 1 == NS ? 0 : cur + 1;
    __builtin_amdgcn_sched_barrier(0);
    read_part(cur, 1, 0, 1);
    mfma_rows(0, 0, FM);
    sched_interleave<FM * FN, FM + FN>();
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(vmcnt_imm((NS - 2) * CPW));
    if (tail && t + 2 == ns) clear_tail(nxt);
    __syncthreads();
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (FM >= 8) {
      // The copies in two bursts, each once the matrix instructions have work.
      constexpr int R0 = FM / 2, NR = FM / 2 + FN / 2;
      mfma_rows(1, 0, 1);
      __builtin_amdgcn_sched_barrier(0);
      issue_a(t + NS, cur);
      read_part(nxt, 0, 0, 2);
      mfma_rows(1, 1, R0);
      sched_interleave<(R0 - 1) * FN, NR>();
      __builtin_amdgcn_sched_barrier(0);
      mfma_rows(1, R0, R0 + 1);
      __builtin_amdgcn_sched_barrier(0);
      issue_b(t + NS, cur);
      read_part(nxt, 0, 1, 2);
      mfma_rows(1, R0 + 1, FM);
      sched_interleave<(FM - R0 - 1) * FN, NR>();
    } else {
      issue_a(t + NS, cur);
      issue_b(t + NS, cur);
      read_part(nxt, 0, 0, 1);
      mfma_rows(1, 0, FM);
      sched_interleave<FM * FN, FM + FN>();
    }
    cur = nxt;
  }
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
  __syncthreads();  // no copy is under way and all waves are done with the stages: the epilogue takes their place
  constexpr int LP = BN + 4;
  float *stg = reinterpret_cast<float *>(smem), *sa = reinterpret_cast<float *>(smem + EPI), *sb = sa + BM;
#pragma unroll
  for (int i = 0; i < SPT; ++i)
    if (threadIdx.x + i * NT < BM + BN) sa[threadIdx.x + i * NT] = scale[i];
  store_tile_passes<BM, BN, WM, WN>(p, m0, n0, 0, stg, [&](int f) {
    const float4_t s = *reinterpret_cast<const float4_t *>(sa + (wm * FM + f) * 16 + 4 * g);
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int col = (wn * FN + j) * 16 + r;
#pragma unroll
      for (int e = 0; e < 4; ++e) stg[(wm * 16 + 4 * g + e) * LP + col] = (float)acc[f][j][e] * sb[col] * s[e];
    }
  });
}

unsigned grid_of(long n, long per) { return (unsigned)std::max(1L, std::min((n + per - 1) / per, 1L << 20)); }

template <int MF, int NF, int KW, int D>
void launch_rows(const Int8Params &p, hipStream_t s) {
  const dim3 grid((unsigned)((p.N + 16 * NF - 1) / (16 * NF)), (unsigned)((p.M + 16 * MF - 1) / (16 * MF)));
  hipLaunchKernelGGL((i8_rows_kernel<MF, NF, KW, D>), grid, dim3(KW * 64), 0, s, p);
}

template <int WM, int WN, int FM, int FN, int NS, int WPE>
void launch_tiles(Int8Params p, hipStream_t s) {
  constexpr int BM = WM * FM * 16, BN = WN * FN * 16;
  p.tiles_m = (int)((p.M + BM - 1) / BM);
  p.tiles_n = (int)((p.N + BN - 1) / BN);
  hipLaunchKernelGGL((i8_tile_kernel<WM, WN, FM, FN, NS, WPE>), dim3((unsigned)(p.tiles_m * p.tiles_n)), dim3(WM * WN * 64), 0, s, p);
}

}  // namespace

int check_int8_gemm(const Int8GemmDesc &d, CError *err) {
  size_t n;
  if (d.K > kInt8MaxK) return set_error(err, -1, "int8 gemm: K of %ld is too large", d.K);
  if (d.M < 0 || d.N < 0 || d.K < 0) return set_error(err, -1, "int8 gemm: negative size");
  // A launch has below 2^32 work-items; up to 512 of them take 16 columns, 256 take 64 rows.
  if (d.M > kMaxRows || d.N > kMaxRows) return set_error(err, -1, "int8 gemm: %ld x %ld is too large", d.M, d.N);
  if (!act_supported(d.act)) return set_error(err, -1, "int8 gemm: unsupported activation %d", d.act);
  if (d.M == 0 || d.N == 0) return 0;
  if (!d.C) return set_error(err, -1, "int8 gemm: NULL C");
  if (d.ldc < d.N) return set_error(err, -1, "int8 gemm: leading dimension smaller than row length");
  if ((uintptr_t)d.C % 4 || (uintptr_t)d.bias % 4 || (uintptr_t)d.a_scales % 4 || (uintptr_t)d.b_scales % 4)
    return set_error(err, -1, "int8 gemm: C, bias or scales not aligned to fp32");
  if (!matrix_bytes(d.M, d.ldc, 4, &n) || n > ((size_t)1 << 62) || (d.M + 15) / 16 > (1L << 26) / ((d.N + 15) / 16))
    return set_error(err, -1, "int8 gemm: problem too large for the grid");
  if (d.K == 0) return 0;
  for (int i = 0; i < 2; ++i) {
    const char *what = i ? "B" : "A";
    const int8_t *x = i ? d.B : d.A;
    const long rows = i ? d.N : d.M, ld = i ? d.ldb : d.lda;
    if (!x) return set_error(err, -1, "int8 gemm: NULL %s", what);
    if (rows > 1 && ld < d.K) return set_error(err, -1, "int8 gemm: leading dimension %ld of %s smaller than row length %ld", ld, what, d.K);
    if ((uintptr_t)x % 16 || (rows > 1 && ld % 16))
      return set_error(err, -1, "int8 gemm: rows of %s at multiples of 16 bytes are needed", what);
    if (rows > 1 && ld > kMaxLd) return set_error(err, -1, "int8 gemm: leading dimension %ld of %s is too large", ld, what);
  }
  return 0;
}

int launch_int8_gemm(const Int8GemmDesc &d, hipStream_t s, CError *err) {
  if (d.M == 0 || d.N == 0) return 0;
  Int8Params p{};
  p.A = d.A;
  p.as = d.a_scales;
  p.B = d.B;
  p.bs = d.b_scales;
  p.C = d.C;
  p.bias = d.bias;
  p.M = d.M, p.N = d.N, p.K = d.K, p.ldc = d.ldc;
  p.lda = d.M > 1 ? d.lda : 0;
  p.ldb = d.N > 1 ? d.ldb : 0;
  p.alpha = d.alpha, p.beta = d.beta, p.act = d.act, p.act_alpha = d.act_alpha;
  if (d.K == 0) {
    hipLaunchKernelGGL(i8_k0_kernel, dim3(grid_of(d.M * d.N, 256)), dim3(256), 0, s, p);
  } else if (d.M <= 16) {
    launch_rows<1, 1, 8, 2>(p, s);
  } else if (d.M <= 64) {
    launch_rows<4, 1, 8, 1>(p, s);
  } else if (d.M * d.N >= 256L * 256 * 200) {
    launch_tiles<2, 4, 8, 4, 2, 2>(p, s);
  } else {
    launch_tiles<2, 2, 4, 4, 2, 2>(p, s);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : hip_error(err, -6, "int8 gemm launch", e);
}

size_t int8_linear_workspace(long M, long N, long K) {
  size_t n;
  if (M < 1 || N < 1 || K < 1 || K > kInt8MaxK || !matrix_bytes(M, int8_pitch(K) + 4, 1, &n)) return 0;
  return (n + 15) / 16 * 16;
}

int check_int8_linear(const Int8LinearDesc &d, CError *err) {
  Int8GemmDesc g = d.gemm;
  if (int rc = check_int8_gemm(Int8GemmDesc{g.M, g.N, 0, g.alpha, g.beta, nullptr, 0, nullptr, nullptr, 0, g.b_scales, g.C, g.ldc, g.bias,
                                            g.act, g.act_alpha}, err))
    return rc;
  const size_t need = int8_linear_workspace(g.M, g.N, g.K);
  // Addresses of the workspace's parts stand in for A's here: sizes, B and the activations are looked at first.
  g.A = reinterpret_cast<const int8_t *>((uintptr_t)16);
  g.lda = int8_pitch(g.K > 0 ? g.K : 0);
  g.a_scales = nullptr;
  if (int rc = check_int8_gemm(g, err)) return rc;
  if (g.M == 0 || g.N == 0 || g.K == 0) return 0;
  Int8QuantizeDesc q{d.dtype, d.x, g.M, g.K, d.ldx, d.col_scale, reinterpret_cast<int8_t *>((uintptr_t)16), g.lda,
                     reinterpret_cast<float *>((uintptr_t)16)};
  if (int rc = check_int8_quantize(q, err)) return rc;
  if (need == 0) return 0;
  if (!d.workspace || d.workspace_bytes < need)
    return set_error(err, -1, "int8 linear: a workspace of %zu bytes is needed, got %zu", need, d.workspace ? d.workspace_bytes : 0);
  if ((uintptr_t)d.workspace % 16) return set_error(err, -1, "int8 linear: a workspace at a multiple of 16 bytes is needed");
  return 0;
}

int launch_int8_linear(const Int8LinearDesc &d, hipStream_t s, CError *err) {
  Int8GemmDesc g = d.gemm;
  if (g.M == 0 || g.N == 0) return 0;
  if (g.K == 0) return launch_int8_gemm(g, s, err);
  const long pitch = int8_pitch(g.K);
  auto *q = static_cast<int8_t *>(d.workspace);
  auto *scales = reinterpret_cast<float *>(q + g.M * pitch);
  if (int rc = launch_int8_quantize({d.dtype, d.x, g.M, g.K, d.ldx, d.col_scale, q, pitch, scales}, s, err)) return rc;
  g.A = q;
  g.lda = pitch;
  g.a_scales = scales;
  return launch_int8_gemm(g, s, err);
}

}  // namespace gn
