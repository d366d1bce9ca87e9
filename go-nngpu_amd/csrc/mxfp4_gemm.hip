// mxfp4_gemm.hip — products with MXFP4 weights, C = act(alpha A B^T + beta C + bias).
#include <algorithm>
#include <climits>

#include "gemm_tile.h"
#include "mxfp4.h"

namespace gn {
namespace {

// 256 rows of codes, and of fp16 activations, stay below 2^31 bytes: 32-bit offsets within a tile.
constexpr long kMaxK = 1L << 22, kMaxRows = 1L << 25;

typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef float float16_t __attribute__((ext_vector_type(16)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

struct MxParams : GemmParams {
  const uint8_t *as, *bs;  // scales
  int G;                   // groups to a row
};

// c + A B^T of 16 x 128 codes each; the scales are byte S of sa and sb.
template <int S>
__device__ __forceinline__ float4_t mfma_fp4(u32x4_t a, u32x4_t b, float4_t c, uint32_t sa, uint32_t sb) {
  const i32x8_t x = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  const i32x8_t y = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 4, 4, S, (int)sa, S, (int)sb);
}

struct __attribute__((packed, aligned(2))) UnalignedHalf8 {
  half8_t v;  // the hardware takes vectors at any address that is a multiple of 2
};

// Eight codes as halves, times 2^(exponent of unit - 127).
__device__ __forceinline__ half8_t half8_of(uint32_t w, float unit) {
  const half2_t a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, unit, 0);
  const half2_t b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, unit, 1);
  const half2_t c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, unit, 2);
  const half2_t d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, unit, 3);
  return half8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Where a scale would take the weights out of fp16's range, the products go through bf16, whose range is fp32's, and an fp16
// number is exactly the sum of two. A code times 2^(E - 127) is a bf16 number for E up to 252; the weights are taken as a quarter
// and the activations (the products' other side, 2^18 at most) four times as large, which serves E up to 254. Twice the
// matrix instructions, the same accumulators, every product still exact.
// A quarter's exponent is below the conversion's range for E of 0 and 1. Such a value is a multiple of 2^-133 below 2^-125, whose
// bits in bf16 are that multiple; the bits of the multiples of 2^-24 in fp16 are the same, and its conversion reaches them.
__device__ __forceinline__ bf16x8_t bf16x8_of(uint32_t w, unsigned e) {
  const bool least = e < 2;
  const float unit = __uint_as_float((least ? e + 107 : e - 2) << 23);  // least: code 2^(E + 4) 2^-24
  u32x4_t v;
  auto pair = [&](bf16x2_t a, half2_t b) { return least ? __builtin_bit_cast(uint32_t, b) : __builtin_bit_cast(uint32_t, a); };
  v[0] = pair(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, unit, 0), __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, unit, 0));
  v[1] = pair(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, unit, 1), __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, unit, 1));
  v[2] = pair(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, unit, 2), __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, unit, 2));
  v[3] = pair(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, unit, 3), __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, unit, 3));
  const u32x4_t nan = {0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};
  return __builtin_bit_cast(bf16x8_t, e == 255 ? nan : v);
}
// c + A B^T of an fp16 A, as the upper 8 bits of 4 A and the rest (0 for infinities and NaN), and of quarters in B.
__device__ __forceinline__ float4_t mfma_halves_bf16(half8_t a, bf16x8_t b, float4_t c) {
  u32x4_t hi, lo;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float x = fmaf((float)a[2 * i], 4.0f, 0.0f), y = fmaf((float)a[2 * i + 1], 4.0f, 0.0f);  // one instruction each
    const uint32_t xh = __float_as_uint(x) & 0xffff0000u, yh = __float_as_uint(y) & 0xffff0000u;
    const float xl = copysignf(fmaxf(fabsf(x - __uint_as_float(xh)), 0.0f), x);  // NaN to 0
    const float yl = copysignf(fmaxf(fabsf(y - __uint_as_float(yh)), 0.0f), y);
    hi[i] = xh >> 16 | yh;
    lo[i] = __float_as_uint(xl) >> 16 | (__float_as_uint(yl) & 0xffff0000u);
  }
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, hi), b, c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, lo), b, c, 0, 0, 0);
}

__device__ __forceinline__ float finish(const MxParams &p, float acc, long m, long n) {
  float v = p.alpha * acc;
  if (p.beta != 0.0f) v += p.beta * p.C[m * p.ldc + n];
  if (p.bias) v += p.bias[n];
  return apply_act(p.act, v, p.act_alpha);
}

// ------------------------------------------------------------------ few rows
// Up to 64 rows: B is read once (1 row 4096 -> 11008: 24 MB, 4.4 us at the rate of reads, in 9.0 us with the launch), and the time
// is that of the loads' latencies, which only in part pass side by side (below). A workgroup owns some columns for all rows;
// its waves cut K among them, whole groups each, and the partial sums meet in LDS. Lane (r, g) = (lane % 16, lane / 16) takes
// block g of row r's group, 16 consecutive bytes, so a wave reads whole 64-byte pieces of 16 rows of B, straight into registers.

// Adds the waves' partial sums and writes C: `part` holds [wk][blocks][64] of them, each block 16 x 16, block j MF + i the
// rows m0 + 16 i .. and the columns n0 + 16 j ... Lane (r, g) of a block has rows 4 g .. 4 g + 3 of column r.
template <int MF>
__device__ __forceinline__ void join_rows(const MxParams &p, const float4_t *part, int wk, int blocks, long m0, long n0) {
  const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6, lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  for (int f = wave; f < blocks; f += waves) {
    float4_t v = part[f * 64 + lane];
    for (int w = 1; w < wk; ++w) v += part[(w * blocks + f) * 64 + lane];
    const long n = n0 + 16 * (f / MF) + r;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const long m = m0 + 16 * (f % MF) + 4 * g + e;
      if (m < p.M && n < p.N) p.C[m * p.ldc + n] = finish(p, v[e], m, n);
    }
  }
}

// Both sides in 4 bits, U groups of NF columns' and MF rows' fragments to a turn. In <1, 1, 4> a turn's loads leave together; of
// the other forms' the compiler moves some to their use, in <2, 4, 2> a column's codes and scales after the first one's, each with
// a wait of its own (16, 32 and 64 rows of 4096 -> 11008 12.2, 16.2 and 19.1 us, the bytes 5 to 6).
template <int MF, int NF, int U>
__global__ void __launch_bounds__(512) mx_fp4_rows_kernel(MxParams p) {
  extern __shared__ float4_t part[];  // [waves][MF * NF][64]
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const long n0 = (long)blockIdx.x * 16 * NF, m0 = (long)blockIdx.y * 16 * MF;
  const int c0 = (int)((long)p.G * wave / waves), c1 = (int)((long)p.G * (wave + 1) / waves);
  float4_t acc[NF][MF];
#pragma unroll
  for (int j = 0; j < NF; ++j)
#pragma unroll
    for (int i = 0; i < MF; ++i) acc[j][i] = float4_t{0.f, 0.f, 0.f, 0.f};
  for (int c = c0; c < c1; c += U) {
    u32x4_t bq[U][NF], aq[U][MF];
    uint32_t bsc[U][NF], asc[U][MF];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long cu = min(c + u, c1 - 1);  // past the wave's last group: that one again, not used
#pragma unroll
      for (int j = 0; j < NF; ++j) {
        const long i = min(n0 + 16 * j + r, p.N - 1) * p.G + cu;
        bq[u][j] = static_cast<const u32x4_t *>(p.B)[i * 4 + g];
        bsc[u][j] = reinterpret_cast<const uint32_t *>(p.bs)[i];
      }
#pragma unroll
      for (int j = 0; j < MF; ++j) {
        const long i = min(m0 + 16 * j + r, p.M - 1) * p.G + cu;
        aq[u][j] = static_cast<const u32x4_t *>(p.A)[i * 4 + g];
        asc[u][j] = reinterpret_cast<const uint32_t *>(p.as)[i];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c + u < c1) {
#pragma unroll
        for (int j = 0; j < NF; ++j)
#pragma unroll
          for (int i = 0; i < MF; ++i)
            acc[j][i] = mfma_fp4<0>(aq[u][i], bq[u][j], acc[j][i], asc[u][i] >> (8 * g), bsc[u][j] >> (8 * g));
      }
  }
#pragma unroll
  for (int j = 0; j < NF; ++j)
#pragma unroll
    for (int i = 0; i < MF; ++i) part[(wave * MF * NF + j * MF + i) * 64 + lane] = acc[j][i];
  __syncthreads();
  join_rows<MF>(p, part, waves, MF * NF, m0, n0);
}

// fp16 activations. K goes in slabs of KS = 128 U WK values, a slab of all rows staged in LDS (through registers: A needs no
// alignment and its tail is masked on the way); WK x WN waves, wave (wk, wn) takes the slab's groups wk U .. wk U + U - 1 and
// NF blocks of columns. The next slab's A and B are asked for before one is multiplied; on their way meanwhile they are for every
// other slab only: behind the branches for A's tail the compiler has no count of the loads, and for the rest it waits for all of
// them before the products (with 17 rows and more for A's chunks one after the other, too). The lane's 32 weights become
// four fragments of v_mfma_f32_16x16x32_f16 whose k are 8 j .. 8 j + 7 of each lane's own block, and A's lanes read the same.
// Where the scales of a wave's blocks all keep the weights normal fp16 numbers (half_exact; weights of ordinary size do) the
// conversion applies them, exactly; otherwise both sides go through bf16.
// Read from the caches by every wave instead of through LDS, A took as long as B and more (4096 -> 11008, fp16 against
// 4-bit activations: 1 row 12.4 against 9.7 us, 16 rows 20 against 14, 64 rows 42 against 25).
// R: the rows of LDS that there may be, 16 MF or fewer.
template <int R, int MF, int NF, int U, int WK, int WN>
__global__ void __launch_bounds__(WK * WN * 64) mx_half_rows_kernel(MxParams p, int lds_rows) {
  constexpr int KS = 128 * U * WK, PITCH = KS + 8;  // halves; the rows of a fragment read start on distinct banks
  constexpr int NT = WK * WN * 64, CPT = R * (KS / 8) / NT;  // 16-byte chunks of a slab to a thread
  extern __shared__ _Float16 slab[];  // [lds_rows][PITCH]; at the end the partial sums
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), wk = wave / WN, wn = wave % WN;
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const long n0 = ((long)blockIdx.x * WN + wn) * 16 * NF, m0 = (long)blockIdx.y * 16 * MF;
  const int ns = (int)((p.K + KS - 1) / KS);

  half8_t st[CPT];
  auto load_slab = [&](int s) {
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      const int q = threadIdx.x + i * NT, row = q / (KS / 8);
      const long k = (long)s * KS + q % (KS / 8) * 8, left = p.K - k;
      st[i] = half8_t{0, 0, 0, 0, 0, 0, 0, 0};
      if (row < lds_rows && m0 + row < p.M && left > 0) {
        const _Float16 *a = static_cast<const _Float16 *>(p.A) + (m0 + row) * p.lda + k;
        if (left >= 8) {
          st[i] = reinterpret_cast<const UnalignedHalf8 *>(a)->v;
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e < left) st[i][e] = a[e];
        }
      }
    }
  };
  auto store_slab = [&] {
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      const int q = threadIdx.x + i * NT, row = q / (KS / 8);
      if (row < lds_rows) *reinterpret_cast<half8_t *>(slab + row * PITCH + q % (KS / 8) * 8) = st[i];
    }
  };
  long brow[NF];
#pragma unroll
  for (int j = 0; j < NF; ++j) brow[j] = min(n0 + 16 * j + r, p.N - 1) * p.G;
  u32x4_t bq[2][U][NF];
  uint32_t bsc[2][U][NF];
  auto load_b = [&](int s, int e) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < NF; ++j) {
        const long i = brow[j] + min((s * WK + wk) * U + u, p.G - 1);  // past the last group: that one, against zeros of A
        bq[e][u][j] = static_cast<const u32x4_t *>(p.B)[i * 4 + g];
        bsc[e][u][j] = reinterpret_cast<const uint32_t *>(p.bs)[i];
      }
  };
  float4_t acc[NF][MF];
#pragma unroll
  for (int j = 0; j < NF; ++j)
#pragma unroll
    for (int i = 0; i < MF; ++i) acc[j][i] = float4_t{0.f, 0.f, 0.f, 0.f};
  int arow[MF];
#pragma unroll
  for (int i = 0; i < MF; ++i) arow[i] = min(16 * i + r, lds_rows - 1) * PITCH + wk * U * kGroup + g * kBlock;

  auto multiply = [&](int s, int e) {
    bool exact = true;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < NF; ++j) exact &= half_exact((bsc[e][u][j] >> (8 * g)) & 255);
    const bool plain = __all(exact);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if ((s * WK + wk) * U + u >= p.G) break;
      if (plain) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          half8_t a[MF];
#pragma unroll
          for (int i = 0; i < MF; ++i) a[i] = *reinterpret_cast<const half8_t *>(slab + arow[i] + u * kGroup + 8 * k);
#pragma unroll
          for (int j = 0; j < NF; ++j) {
            const half8_t w = half8_of(bq[e][u][j][k], __uint_as_float(((bsc[e][u][j] >> (8 * g)) & 255) << 23));
#pragma unroll
            for (int i = 0; i < MF; ++i) acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[i], w, acc[j][i], 0, 0, 0);
          }
        }
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int j = 0; j < NF; ++j) {
            const bf16x8_t w = bf16x8_of(bq[e][u][j][k], (bsc[e][u][j] >> (8 * g)) & 255);
#pragma unroll
            for (int i = 0; i < MF; ++i) {
              acc[j][i] = mfma_halves_bf16(*reinterpret_cast<const half8_t *>(slab + arow[i] + u * kGroup + 8 * k), w, acc[j][i]);
              __builtin_amdgcn_sched_barrier(0);  // one product's operands in registers at a time
            }
          }
      }
    }
  };
  // One slab in LDS, the next one's loads under way meanwhile; two slabs to a turn, so that B's registers are named.
  load_b(0, 0);
  load_slab(0);
  for (int s = 0;;) {
    store_slab();
    __syncthreads();
    if (s + 1 < ns) load_b(s + 1, 1), load_slab(s + 1);
    multiply(s, 0);
    __syncthreads();
    if (++s == ns) break;
    store_slab();
    __syncthreads();
    if (s + 1 < ns) load_b(s + 1, 0), load_slab(s + 1);
    multiply(s, 1);
    __syncthreads();
    if (++s == ns) break;
  }
  float4_t *part = reinterpret_cast<float4_t *>(slab);
#pragma unroll
  for (int j = 0; j < NF; ++j)
#pragma unroll
    for (int i = 0; i < MF; ++i) part[(wk * MF * NF * WN + (wn * NF + j) * MF + i) * 64 + lane] = acc[j][i];
  __syncthreads();
  join_rows<MF>(p, part, WK, MF * NF * WN, m0, (long)blockIdx.x * WN * 16 * NF);
}

// K == 0: act(beta C + bias).
__global__ void __launch_bounds__(256) mx_k0_kernel(MxParams p) {
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < p.M * p.N; i += (long)gridDim.x * 256)
    p.C[i / p.N * p.ldc + i % p.N] = finish(p, 0.0f, i / p.N, i % p.N);
}

// ------------------------------------------------------------------ both sides in 4 bits
// c + A B^T of 32 x 64 codes each; the scales are byte S of sa and sb.
template <int S>
__device__ __forceinline__ float16_t mfma32_fp4(u32x4_t a, u32x4_t b, float16_t c, uint32_t sa, uint32_t sb) {
  const i32x8_t x = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  const i32x8_t y = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x, y, c, 4, 4, S, (int)sa, S, (int)sb);
}

// C = A B^T on v_mfma_scale_f32_32x32x64_f8f6f4 (from registers it sustains 6.4 PFLOP/s on random codes and 9.7 on
// zeros, the 16 x 16 x 128 form 5.8 and 6.8). WM x WN waves, each FM x FN blocks of 32 x 32. K goes in stages of
// a group (128 values, 64 bytes of codes to a row), copied straight to LDS by dma16 in chunks of 16 rows,
// kSlots stages in flight. A row's 16 bytes o sit at place o ^ ((row >> 2) & 3) of its 64: the 16 rows that a phase of a
// fragment read touches fall on distinct banks. Lane half h takes block 2 h + s of its row's four in step s of
// two, on both sides, so its scales for the stage are two bytes next to each other, and the instruction's byte
// selector is s. A row's scales for four stages are 16 bytes, copied to LDS by the same means: read into registers by each
// wave they cost one cache line to a row and stage, and with two stages of 256 in flight that bound the kernel
// (8192^3 369 us). A step multiplies while the next one's fragments are read; before a stage's second step the next
// stage has landed (one wait and one barrier to a stage), and the copies of the one kSlots ahead go into the slot just left.
// 8192^3 takes 297 us (3.7 PFLOP/s): the loop goes at 4.7, and some 60 us are the tiles' ends, where all CUs write C at
// once (the matrix units are busy for half of the cycles, waves wait for 38%). Smaller tiles read a fragment of LDS for each
// matrix instruction and are bound by that and by the barriers (512 rows, 4096 -> 11008: 23.7 us; the operations alone 7, C alone 5).
constexpr int kSlots = 4;
template <int WM, int WN, int FM, int FN, int WPE>
__global__ void __launch_bounds__(WM * WN * 64) __attribute__((amdgpu_waves_per_eu(WPE, WPE)))
mx_fp4_kernel(MxParams p) {
  constexpr int NW = WM * WN, BM = WM * FM * 32, BN = WN * FN * 32;
  constexpr int CA = BM / 16 / NW, CB = BN / 16 / NW, CPW = CA + CB;  // chunks of 16 rows to a wave
  constexpr int STAGE = (BM + BN) * 64, SCALES = (BM + BN) * 16;      // bytes; SCALES: of four stages
  constexpr int LDS = kSlots * STAGE + 2 * SCALES, EPI = WM * 16 * (BN + 4) * 4;
  static_assert(CA * NW * 16 == BM && CB * NW * 16 == BN && BM % 64 == 0 && BN % 64 == 0 && kSlots == 4, "chunks");
  __shared__ __attribute__((aligned(1024))) char smem[LDS > EPI ? LDS : EPI];

  int tm, tn;
  tile_coords(p, tm, tn);
  const long m0 = (long)tm * BM, n0 = (long)tn * BN;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wm = wave / WN, wn = wave % WN, l32 = lane & 31, h = lane >> 5;
  const unsigned pitch = 64u * (unsigned)p.G, spitch = 4u * (unsigned)p.G;

  // Codes: lane L of chunk c copies 16 bytes of row 16 c + L / 4, which land at 16 L of the chunk.
  const char *a0 = static_cast<const char *>(p.A) + m0 * pitch, *b0 = static_cast<const char *>(p.B) + n0 * pitch;
  const unsigned oct = 16u * ((lane & 3) ^ ((lane >> 4) & 3));
  unsigned va[CA], vb[CB];
#pragma unroll
  for (int i = 0; i < CA; ++i) {
    const int row = 16 * (wave * CA + i) + (lane >> 2);
    va[i] = m0 + row < p.M ? row * pitch + oct : kOutOfRange;
  }
#pragma unroll
  for (int i = 0; i < CB; ++i) {
    const int row = 16 * (wave * CB + i) + (lane >> 2);
    vb[i] = n0 + row < p.N ? row * pitch + oct : kOutOfRange;
  }
  const unsigned lds = lds_offset(smem);
  auto issue = [&](int t) {  // past the last stage all reads are zeros
    BufRsrc da = make_rsrc(a0 + 64L * t), db = make_rsrc(b0 + 64L * t);
    da.r.z = db.r.z = __builtin_amdgcn_readfirstlane(t < p.G ? (int)ring::kNumRecords : 0);
    const unsigned st = lds + (t & (kSlots - 1)) * STAGE;
#pragma unroll
    for (int i = 0; i < CA; ++i) dma16(da, va[i], __builtin_amdgcn_readfirstlane(st + (wave * CA + i) * 1024));
#pragma unroll
    for (int i = 0; i < CB; ++i) dma16(db, vb[i], __builtin_amdgcn_readfirstlane(st + BM * 64 + (wave * CB + i) * 1024));
  };
  // Scales: wave w copies rows 64 w .. 64 w + 63 of the tile's BM + BN (then 64 (w + NW) ..), 16 bytes of each. Rows past
  // the matrix and bytes past its end are zeros, groups past a row's end are another row's; the stages that they belong to are
  // not run.
  constexpr int SB = (BM + BN) / 64;  // blocks of 64 rows
  auto issue_scales = [&](int c) {  // of stages 4 c .. 4 c + 3
#pragma unroll
    for (int i = 0; i < (SB + NW - 1) / NW; ++i) {
      const int blk = wave + i * NW;
      const bool is_a = blk < BM / 64;
      if (blk >= SB) break;
      const long rows = is_a ? min(p.M - m0, (long)BM) : min(p.N - n0, (long)BN);
      const int row = 64 * (is_a ? blk : blk - BM / 64) + lane;
      BufRsrc ds = make_rsrc((is_a ? p.as : p.bs) + (is_a ? m0 : n0) * spitch);
      ds.r.z = __builtin_amdgcn_readfirstlane((int)(rows * spitch));
      dma16(ds, 4 * c < p.G && row < rows ? row * spitch + 16 * c : kOutOfRange,
            __builtin_amdgcn_readfirstlane(lds + kSlots * STAGE + (c & 1) * SCALES + blk * 1024));
    }
  };

  u32x4_t fa[2][FM], fb[2][FN];   // fragments of even and odd steps
  u32x4_t qa[FM], qb[FN];         // scales of four stages
  const unsigned arow = (wm * FM * 32 + l32) * 64, brow = BM * 64 + (wn * FN * 32 + l32) * 64;
  const unsigned sw = ((2 * h) ^ ((l32 >> 2) & 3)) << 4;
  auto read_frags = [&](int t, int s) {
    const char *st = smem + (t & (kSlots - 1)) * STAGE + (sw ^ (s << 4));
#pragma unroll
    for (int i = 0; i < FM; ++i) fa[s][i] = *reinterpret_cast<const u32x4_t *>(st + arow + i * 2048);
#pragma unroll
    for (int i = 0; i < FN; ++i) fb[s][i] = *reinterpret_cast<const u32x4_t *>(st + brow + i * 2048);
  };
  auto read_scales = [&](int t) {  // of stages t .. t + 3
    const char *st = smem + kSlots * STAGE + ((t >> 2) & 1) * SCALES + l32 * 16;
#pragma unroll
    for (int i = 0; i < FM; ++i) qa[i] = *reinterpret_cast<const u32x4_t *>(st + (wm * FM + i) * 512);
#pragma unroll
    for (int i = 0; i < FN; ++i) qb[i] = *reinterpret_cast<const u32x4_t *>(st + (BM + (wn * FN + i) * 32) * 16);
  };
  // Stage s of the four: a lane's two bytes to the low end.
  uint32_t ca[FM], cb[FN];
  auto take_scales = [&](int s) {
#pragma unroll
    for (int i = 0; i < FM; ++i) ca[i] = qa[i][s] >> (16 * h);
#pragma unroll
    for (int i = 0; i < FN; ++i) cb[i] = qb[i][s] >> (16 * h);
  };
  float16_t acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  auto mfma_rows = [&](auto step, int i0, int i1) {
    constexpr int S = decltype(step)::value;
#pragma unroll
    for (int i = 0; i < FM; ++i)
      if (i >= i0 && i < i1)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = mfma32_fp4<S>(fa[S][i], fb[S][j], acc[i][j], ca[i], cb[j]);
  };
  auto stage = [&](int t, auto of) {
    constexpr int Q = decltype(of)::value;  // t % 4
    __builtin_amdgcn_sched_barrier(0);
    read_frags(t, 1);
    take_scales(Q);
    mfma_rows(ActCode<0>{}, 0, FM);
    sched_interleave<FM * FN, FM + FN>();
    __builtin_amdgcn_sched_barrier(0);
    // All but the copies of stages t + 2 and t + 3 (and scales between them) are done: stage t + 1 is there.
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(2 * CPW));
    __syncthreads();
    __builtin_amdgcn_sched_barrier(0);
    mfma_rows(ActCode<1>{}, 0, 1);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (Q == 0) issue_scales(t / 4 + 1);  // before stage t + 4's codes: there when they are
    issue(t + kSlots);
    read_frags(t + 1, 0);  // past the last stage: zeros, never used
    if constexpr (Q == 3) read_scales(t + 1);
    mfma_rows(ActCode<1>{}, 1, FM);
    sched_interleave<(FM - 1) * FN, FM + FN>();
  };

  issue_scales(0);
#pragma unroll
  for (int t = 0; t < kSlots; ++t) issue(t);
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(3 * CPW));
  __syncthreads();
  read_frags(0, 0);
  read_scales(0);
  for (int t = 0;;) {
    stage(t, ActCode<0>{});
    if (++t == p.G) break;
    stage(t, ActCode<1>{});
    if (++t == p.G) break;
    stage(t, ActCode<2>{});
    if (++t == p.G) break;
    stage(t, ActCode<3>{});
    if (++t == p.G) break;
  }
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
  __syncthreads();  // no copy is under way and all waves are done with the slots: the epilogue takes their place
  // Block (i, j): register r of lane (l32, h) holds row 8 (r / 4) + 4 h + r % 4 of column l32.
  constexpr int LP = BN + 4;
  float *stg = reinterpret_cast<float *>(smem);
  store_tile_passes<BM, BN, WM, WN>(p, m0, n0, 0, stg, [&](int f) {
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int r = 0; r < 8; ++r)
        stg[(wm * 16 + 8 * (r / 4) + 4 * h + r % 4) * LP + (wn * FN + j) * 32 + l32] = acc[f / 2][j][8 * (f & 1) + r];
  });
}

// ------------------------------------------------------------------ fp16 activations, many rows
// C = A B^T on v_mfma_f32_16x16x32_f16, the weights converted in registers. WM x WN waves, each FM x FN blocks of 16 x 16;
// K in stages of 64, NS of them in LDS: 128 bytes of A to a row (ring_plan.h's plan and swizzle) and 32 of codes. Lane (r,
// g) takes k = 16 g .. 16 g + 15 of the stage on both sides, 8 in each of two steps, so its 16 codes are 8 consecutive bytes (a
// wave's read of 16 rows is 512 consecutive ones) and lie in one block. A row's scales for 8 stages are 16 bytes in LDS. A tile's
// weights are applied in fp16 where all of its columns' scales allow it over the whole of K, else in bf16, at 3.4 times the time
// and, but for the 256 x 256 tile, after a pass in fp16 that is thrown away: with one block in 32 rows of B out of
// range, as a pruned layer may have them (a largest weight below 2^-21), 128 rows 4096 -> 11008 105 us instead of 24, 512 rows 203
// instead of 52, 8192^3 2.81 ms instead of 0.83. (In the few-rows kernel a wave decides for each of its slabs: 64 rows 29 instead of 26 us.)
// 8192^3 takes 820 us (1.34 PFLOP/s, the rate of a large bf16 library product on this card: its power); smaller products wait for LDS and
// the barriers between stages (128 x 128 tiles without their matrix instructions took 85% of their time, without their copies 75%).
// DMA: A is copied to LDS by dma16 (16-byte aligned rows, K a multiple of 8); otherwise through registers, its tail masked.
template <int WM, int WN, int FM, int FN, int NS>
struct HalfTile {
  static constexpr int BM = WM * FM * 16, BN = WN * FN * 16;
  static constexpr int STAGE = BM * 128 + BN * 32, SCALES = BN * 16, SPARE = BN / 32 % (WM * WN) ? 1024 : 0;
  static constexpr int LDS = NS * STAGE + 2 * SCALES + SPARE, EPI = WM * 16 * (BN + 4) * 4;
  static constexpr int BYTES = LDS > EPI ? LDS : EPI;
};

// The tile in fp16 (PLAIN) or bf16. With CHECK it looks at its scales on the way, and returns with nothing written where fp16
// did not do; otherwise the wave ends. A branch to the other form in each stage, or after the first one that needs it, had the
// compiler move all accumulators between registers (4096 -> 11008, 512 rows: 72 us against 63).
template <int WM, int WN, int FM, int FN, int NS, bool DMA, bool PLAIN, bool CHECK>
__device__ __forceinline__ void half_tile(const MxParams &p, char *smem, int tm, int tn, int tid) {
  constexpr int NW = WM * WN, BM = WM * FM * 16, BN = WN * FN * 16;
  constexpr int CA = BM / 8 / NW, NB = BN / 32, CB = (NB + NW - 1) / NW;  // 1 KiB chunks of A to a wave; of B, and to a wave
  constexpr int SB = BN / 64;
  using Tile = HalfTile<WM, WN, FM, FN, NS>;
  constexpr int STAGE = Tile::STAGE, SCALES = Tile::SCALES, LDS = Tile::LDS;
  static_assert(CA * NW * 8 == BM && CA % 2 == 0 && BN % 64 == 0 && SB <= NW, "chunks");
  const long m0 = (long)tm * BM, n0 = (long)tn * BN;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int wm = wave / WN, wn = wave % WN, r = lane & 15, g = lane >> 4;
  const unsigned pitch = 64u * (unsigned)p.G, spitch = 4u * (unsigned)p.G;
  const int ns = (int)((p.K + 63) / 64);
  const unsigned lds = lds_offset(smem);

  // A: lane L of chunk c copies octet kc8_octet(row, L & 7) of row 8 c + L / 8.
  const char *a0 = static_cast<const char *>(p.A) + m0 * p.lda * 2, *b0 = static_cast<const char *>(p.B) + n0 * pitch;
  unsigned va[CA], vb[CB];
  // The copy's first k in the stage, for even i; for odd i the octet's upper bit is the other way round (row >> 1 is 4 more).
  const int ka = 8 * kc8_octet(8 * wave * CA + (lane >> 3), lane & 7);
  auto k_of = [&](int i) { return ka ^ (i & 1 ? 32 : 0); };
#pragma unroll
  for (int i = 0; i < CA; ++i) {
    const int row = 8 * (wave * CA + i) + (lane >> 3), o = kc8_octet(row, lane & 7);
    va[i] = m0 + row < p.M ? (unsigned)(row * p.lda * 2 + 16 * o) : kOutOfRange;
  }
#pragma unroll
  for (int i = 0; i < CB; ++i) {
    const int row = 32 * (wave + i * NW) + (lane >> 1);
    // A wave without a chunk copies zeros to a place of its own: every wave has as many copies in flight.
    vb[i] = row < BN && n0 + row < p.N ? row * pitch + 16 * (lane & 1) : kOutOfRange;
  }
  auto issue = [&](int t, unsigned slot) {  // past the last stage all reads are zeros
    const int left = (int)p.K - 64 * t;
    const unsigned st = lds + slot;
    if constexpr (DMA) {
      BufRsrc da = make_rsrc(a0 + 128L * t);
      if (left >= 64) {
#pragma unroll
        for (int i = 0; i < CA; ++i) dma16(da, va[i], __builtin_amdgcn_readfirstlane(st + (wave * CA + i) * 1024));
      } else {
#pragma unroll
        for (int i = 0; i < CA; ++i)
          dma16(da, k_of(i) < left ? va[i] : kOutOfRange, __builtin_amdgcn_readfirstlane(st + (wave * CA + i) * 1024));
      }
    }
    BufRsrc db = make_rsrc(b0 + 32L * t);
    db.r.z = __builtin_amdgcn_readfirstlane(left > 0 ? (int)ring::kNumRecords : 0);
#pragma unroll
    for (int i = 0; i < CB; ++i)
      dma16(db, vb[i], __builtin_amdgcn_readfirstlane(wave + i * NW < NB ? st + BM * 128 + (wave + i * NW) * 1024 : lds + LDS - 1024));
  };
  half8_t ar[DMA ? 1 : CA];
  auto load_a = [&](int t) {  // A's part of issue(), to registers
    const long left = p.K - 64L * t;
#pragma unroll
    for (int i = 0; i < CA; ++i) {
      ar[DMA ? 0 : i] = half8_t{0, 0, 0, 0, 0, 0, 0, 0};
      const _Float16 *a = reinterpret_cast<const _Float16 *>(a0 + 128L * t + va[i]);
      if (va[i] != kOutOfRange) {
        if (k_of(i) + 8 <= left) {
          ar[DMA ? 0 : i] = reinterpret_cast<const UnalignedHalf8 *>(a)->v;
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (k_of(i) + e < left) ar[DMA ? 0 : i][e] = a[e];
        }
      }
    }
  };
  auto store_a = [&](unsigned slot) {
    char *st = smem + slot;
#pragma unroll
    for (int i = 0; i < CA; ++i) *reinterpret_cast<half8_t *>(st + (wave * CA + i) * 1024 + lane * 16) = ar[DMA ? 0 : i];
  };
  const long s_rows = min(p.N - n0, (long)BN);
  auto issue_scales = [&](int c) {  // of stages 8 c .. 8 c + 7; bytes past a row's end are another row's, not used
    if (wave < SB) {
      const int row = min(64 * wave + lane, (int)s_rows - 1);  // past the matrix the last row's, against zeros
      BufRsrc ds = make_rsrc(p.bs + n0 * spitch);
      ds.r.z = __builtin_amdgcn_readfirstlane((int)(s_rows * spitch));
      dma16(ds, 4 * c < p.G ? row * spitch + 16 * c : kOutOfRange,
            __builtin_amdgcn_readfirstlane(lds + NS * STAGE + (c & 1) * SCALES + wave * 1024));
    }
  };

  half8_t fa[FM];
  u32x2_t bq[FN];
  unsigned be[FN];  // scale bytes
  const unsigned arow = (wm * FM * 16 + r) * 128, asw = (2 * g) ^ ((r >> 1) & 7);
  auto read_a = [&](unsigned slot, int s, int i) {
    return *reinterpret_cast<const half8_t *>(smem + slot + arow + i * 2048 + ((asw ^ s) << 4));
  };
  auto scale_at = [&](int t, int j) {
    return smem + NS * STAGE + ((t >> 3) & 1) * SCALES + ((wn * FN + j) * 16 + r) * 16 + 2 * (t & 7);
  };
  auto read_b = [&](int t, unsigned slot) {
    const char *st = smem + slot + BM * 128 + (wn * FN * 16 + r) * 32 + 8 * g;
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      bq[j] = *reinterpret_cast<const u32x2_t *>(st + j * 512);
      be[j] = *reinterpret_cast<const uint8_t *>(scale_at(t, j) + (g >> 1));
    }
  };
  float4_t acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = float4_t{0.f, 0.f, 0.f, 0.f};

  // The step's products, row by row; each fragment of A is read anew, into the same registers, once it has been used. In fp16
  // the other step's weights are converted on the way (from row `from` on), in bf16 this one's before.
  u32x4_t w[PLAIN ? 2 : 1][FN];
  unsigned worst = 0;  // above the width of half_exact's range if a scale was outside of it
  auto check = [&] {
#pragma unroll
    for (int j = 0; j < FN; ++j) worst = max(worst, be[j] - kHalfLeast);
  };
  auto weight = [&](int s, int j) {
    if constexpr (PLAIN)
      w[s][j] = __builtin_bit_cast(u32x4_t, half8_of(bq[j][s], __uint_as_float(be[j] << 23)));
    else
      w[0][j] = __builtin_bit_cast(u32x4_t, bf16x8_of(bq[j][s], be[j]));
  };
  auto multiply = [&](auto step, unsigned slot, int from, auto after_first) {
    constexpr int S = decltype(step)::value;
    if constexpr (!PLAIN) {
#pragma unroll
      for (int j = 0; j < FN; ++j) weight(S, j);
    }
#pragma unroll
    for (int i = 0; i < FM; ++i) {
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        if constexpr (PLAIN) {
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fa[i], __builtin_bit_cast(half8_t, w[S][j]), acc[i][j], 0, 0, 0);
        } else {
          acc[i][j] = mfma_halves_bf16(fa[i], __builtin_bit_cast(bf16x8_t, w[0][j]), acc[i][j]);
          __builtin_amdgcn_sched_barrier(0);  // one product's operands in registers at a time
        }
      }
      fa[i] = read_a(slot, 1 - S, i);
      if constexpr (PLAIN) {
#pragma unroll
        for (int j = 0; j < FN; ++j)
          if (from + j * (FM - from) / FN == i) weight(1 - S, j);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (i == 0) after_first();
    }
  };

  issue_scales(0);
#pragma unroll
  for (int i = 0; i < NS; ++i) issue(i, i * STAGE);
  if constexpr (!DMA) {
#pragma unroll
    for (int i = 0; i < NS - 1; ++i) {
      load_a(i);
      store_a(i * STAGE);
    }
    load_a(NS - 1);
  }
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
  __syncthreads();
  read_b(0, 0);
#pragma unroll
  for (int i = 0; i < FM; ++i) fa[i] = read_a(0, 0, i);
  if constexpr (PLAIN) {
#pragma unroll
    for (int j = 0; j < FN; ++j) weight(0, j);
  }
  auto stage = [&](int t, unsigned here, unsigned next, unsigned before) {  // the slots of stages t, t + 1 and t - 1
    if constexpr (CHECK) check();
    multiply(ActCode<0>{}, here, 0, [] {});
    // All but the copies of stage t + 2 and later are done: stage t + 1 is there.
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(DMA ? (NS - 2) * (CA + CB) : 0));
    __syncthreads();
    auto copies = [&] {
      if ((t & 7) == 0) issue_scales(t / 8 + 1);
      if constexpr (!DMA) {
        store_a(before);
        load_a(t + NS);
      }
      issue(t + NS, here);
    };
    // The copies once the matrix instructions have work, where there are registers for it.
    constexpr bool kLate = FM * FN < 32;
    if constexpr (!kLate) copies();
    // Past the last stage zeros, and scales that are not looked at.
    if constexpr (PLAIN) read_b(t + 1, next);
    multiply(ActCode<1>{}, next, FM / 2, [&] {
      if constexpr (kLate) copies();
    });
    if constexpr (!PLAIN) read_b(t + 1, next);
  };
  // Slots that the compiler knows save a third of the scalar instructions, which such tiles wait for (128 rows 4096 -> 11008 26.1
  // instead of 30.9 us; 512 rows 11008 -> 4096 57.5, 68.6); the 256 x 256 tile does not (8192^3 847 instead of 827).
  if constexpr (FM * FN < 32) {
    for (int t = 0;;) {
      stage(t, 0, STAGE, (NS - 1) * STAGE);
      if (++t == ns) break;
      stage(t, STAGE, 2 * STAGE, 0);
      if (++t == ns) break;
      stage(t, 2 * STAGE, 3 % NS * STAGE, STAGE);
      if (++t == ns) break;
      if constexpr (NS == 4) {
        stage(t, 3 * STAGE, 0, 2 * STAGE);
        if (++t == ns) break;
      }
    }
  } else {
    unsigned here = 0, before = (NS - 1) * STAGE;
    for (int t = 0; t < ns; ++t) {
      const unsigned next = here == (NS - 1) * STAGE ? 0 : here + STAGE;
      stage(t, here, next, before);
      before = here, here = next;
    }
  }
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
  // No copy is under way and all waves are done with the slots: the epilogue takes their place.
  if constexpr (CHECK) {
    if (__builtin_amdgcn_readfirstlane(__syncthreads_or(worst > kHalfWidth))) return;
  } else {
    __syncthreads();
  }
  // What only the epilogue needs of the arguments is read again: kept through the loop it takes scalar registers that the loop has not.
  auto *args = (const CONST_AS MxParams *)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(args));
  const MxParams e = *(const MxParams *)args;
  store_tile_rows<BM, BN, WM, WN>(e, m0, n0, 0, reinterpret_cast<float *>(smem), acc);
  if constexpr (CHECK) __builtin_amdgcn_endpgm();
}

// Whether fp16 does for the columns of a tile: all their scales, which lie one after the other.
template <int NT, int BN>
__device__ __forceinline__ bool scan_scales(const MxParams &p, int tn) {
  const long n0 = (long)tn * BN, count = min(p.N - n0, (long)BN) * p.G;
  const uint32_t *s = reinterpret_cast<const uint32_t *>(p.bs) + n0 * p.G;
  bool fits = true;
#pragma unroll 8
  for (long i = threadIdx.x; i < count; i += NT) {
    const uint32_t v = s[i];
#pragma unroll
    for (int k = 0; k < 32; k += 8) fits &= half_exact((v >> k) & 255);
  }
  return !__builtin_amdgcn_readfirstlane(__syncthreads_or(!fits));
}

template <int WM, int WN, int FM, int FN, int NS, int WPE, bool DMA>
__global__ void __launch_bounds__(WM * WN * 64) __attribute__((amdgpu_waves_per_eu(WPE, WPE)))
mx_half_kernel(MxParams p) {
  __shared__ __attribute__((aligned(1024))) char smem[HalfTile<WM, WN, FM, FN, NS>::BYTES];
  int tm, tn;
  tile_coords(p, tm, tn);
  // The tall tile looks at the scales first, 1% of its time: its accumulators leave no registers to keep through the other
  // form's code, as the compiler does where that follows.
  constexpr bool TALL = FM > 4;
  bool fp16 = true;
  if constexpr (TALL) fp16 = scan_scales<WM * WN * 64, HalfTile<WM, WN, FM, FN, NS>::BN>(p, tn);
  if (fp16) {
    half_tile<WM, WN, FM, FN, NS, DMA, true, !TALL>(p, smem, tm, tn, threadIdx.x);
    if constexpr (TALL) return;
  }
  // bf16 takes more registers: a tall tile in two halves, with arguments (the kernel's, p is the only one) and addresses that
  // the compiler does not keep from the first form.
  constexpr int H = TALL ? 2 : 1;
  auto *args = (const CONST_AS MxParams *)__builtin_amdgcn_kernarg_segment_ptr();
  int tid = threadIdx.x;
#pragma unroll 1
  for (int h = 0; h < H; ++h) {
    __syncthreads();
    asm volatile("" : "+v"(tid), "+s"(args));
    const MxParams q = *(const MxParams *)args;
    int um, un;
    tile_coords(q, um, un);
    if ((long)(um * H + h) * (WM * FM / H * 16) < q.M)
      half_tile<WM, WN, FM / H, FN, NS, DMA, false, false>(q, smem, um * H + h, un, tid);
  }
}

unsigned grid_of(long n, long per) { return (unsigned)std::max(1L, std::min((n + per - 1) / per, 1L << 20)); }

template <int WM, int WN, int FM, int FN, int WPE>
void launch_fp4(MxParams p, hipStream_t s) {
  constexpr int BM = WM * FM * 32, BN = WN * FN * 32;
  p.tiles_m = (int)((p.M + BM - 1) / BM);
  p.tiles_n = (int)((p.N + BN - 1) / BN);
  hipLaunchKernelGGL((mx_fp4_kernel<WM, WN, FM, FN, WPE>), dim3((unsigned)(p.tiles_m * p.tiles_n)), dim3(WM * WN * 64), 0, s, p);
}

template <int WM, int WN, int FM, int FN, int NS, int WPE, bool DMA>
void launch_half(MxParams p, hipStream_t s) {
  constexpr int BM = WM * FM * 16, BN = WN * FN * 16;
  p.tiles_m = (int)((p.M + BM - 1) / BM);
  p.tiles_n = (int)((p.N + BN - 1) / BN);
  hipLaunchKernelGGL((mx_half_kernel<WM, WN, FM, FN, NS, WPE, DMA>), dim3((unsigned)(p.tiles_m * p.tiles_n)), dim3(WM * WN * 64), 0, s, p);
}

// More than 64 rows: the kind of tile with which a CU's share takes the least time, the largest one of equals. alone: a stage of
// one tile on a CU, in units of 10 ns, more: of each further one of its share.
struct TileCost {
  int bm, bn, alone, more;
};
int cheapest_tile(const MxParams &p, const TileCost (&kinds)[5]) {
  int best = 0;
  long least = 0;
  for (int i = 0; i < 5; ++i) {
    const TileCost &k = kinds[i];
    const long tiles = ((p.M + k.bm - 1) / k.bm) * ((p.N + k.bn - 1) / k.bn);
    const long cost = k.alone + (tiles - 1) / 256 * k.more;  // 256 CUs
    if (i == 0 || cost < least) best = i, least = cost;
  }
  return best;
}

// 4-bit activations: the largest tile goes at the rate of the matrix instructions, the smallest at the latency of its copies and
// barriers. Measured, us, 256 x 256 / 256 x 128 / 128 x 128 / 64 x 128 / 64 x 64: 4096 -> 11008, 1024 rows 36.6 / 45.9 / 43.0 /
// 50.5 / 63.7, 512 rows 33.3 / 23.7 / 27.8 / 29.6 / 38.8, 200 rows 29.0 / 18.6 / 15.6 / 17.5 / 19.6, 128 rows 28.0 / 18.3 / 15.3 /
// 11.8 / 12.3; 11008 -> 4096, 512 rows 69.9 / 47.1 / 35.1 / 28.0 / 34.2; 4096 -> 4096, 65 rows 26.7 / 17.2 / 13.9 / 11.4 / 9.2.
void launch_fp4_tiles(const MxParams &p, hipStream_t s) {
  constexpr TileCost kTiles[] = {{256, 256, 75, 75}, {256, 128, 50, 50}, {128, 128, 35, 35}, {64, 128, 28, 28}, {64, 64, 20, 20}};
  switch (cheapest_tile(p, kTiles)) {
    case 0: return launch_fp4<2, 4, 4, 2, 2>(p, s);
    case 1: return launch_fp4<4, 2, 2, 2, 2>(p, s);
    case 2: return launch_fp4<2, 2, 2, 2, 2>(p, s);
    case 3: return launch_fp4<2, 2, 1, 2, 2>(p, s);
    default: return launch_fp4<2, 2, 1, 1, 2>(p, s);
  }
}

// The same for fp16 activations; rows of A that are not 16-byte aligned go through registers in 128 x 64 tiles, with a wait for all
// copies in each stage (K of 4097 against 4096, 512 rows -> 11008: 125 against 55 us, 2048 rows -> 4096 130 / 68; 8192 x 8193 -> 8192
// 1.86 / 0.83 ms): a copy with aligned rows would need memory that this call, which allocates nothing, does not have. Two tiles of the
// three smaller kinds share a CU and its time. Measured, us, 256 x 256 / 128 x 192 / 128 x 128 / 64 x 128 / 64 x 64: 8192^3 825 / 1001 /
// 925 / 1073 / 1401; 4096 -> 11008, 1024 rows 111 / 115 / 105 / 114 / 143, 512 rows 98 / 52.6 / 62.8 / 55.6 / 70.8, 256 rows 97 / 46.2 /
// 38.4 / 36.7 / 37.0, 128 rows 96 / 46.0 / 37.6 / 24.6 / 25.7; 4096 -> 4096, 2048 rows 102 / 95 / 67.3 / 74.0 / 90.6, 128 rows 95 /
// 45.6 / 37.6 / 23.5 / 19.8. Waves of 128 x 32 (64 x 64: the weights of a column converted by two waves) took 39 instead of 45 us
// for the 128 x 128 tiles of 128 rows 4096 -> 4096.
void launch_half_tiles(const MxParams &p, hipStream_t s) {
  if ((uintptr_t)p.A % 16 != 0 || p.lda % 8 != 0 || p.K % 8 != 0) return launch_half<2, 2, 4, 2, 3, 2, false>(p, s);
  constexpr TileCost kTiles[] = {{256, 256, 142, 142}, {128, 192, 64, 71}, {128, 128, 55, 38}, {64, 128, 30, 24}, {64, 64, 24, 14}};
  switch (cheapest_tile(p, kTiles)) {
    case 0: return launch_half<2, 4, 8, 4, 3, 2, true>(p, s);
    case 1: return launch_half<2, 4, 4, 3, 4, 2, true>(p, s);
    case 2: return launch_half<1, 4, 8, 2, 3, 2, true>(p, s);
    case 3: return launch_half<1, 4, 4, 2, 4, 3, true>(p, s);
    default: return launch_half<1, 4, 4, 1, 4, 3, true>(p, s);
  }
}

template <int MF, int NF, int U>
void launch_fp4_rows(const MxParams &p, hipStream_t s) {
  int waves = 1;  // as many as give each at most U groups, 8 at most
  while (waves < 8 && waves * U < p.G) waves *= 2;
  const dim3 grid((unsigned)((p.N + 16 * NF - 1) / (16 * NF)), (unsigned)((p.M + 16 * MF - 1) / (16 * MF)));
  hipLaunchKernelGGL((mx_fp4_rows_kernel<MF, NF, U>), grid, dim3(waves * 64), waves * MF * NF * 1024, s, p);
}

template <int R, int MF, int NF, int U, int WK, int WN>
void launch_half_rows(const MxParams &p, hipStream_t s) {
  const int rows = (int)std::min(p.M, (long)R);
  const size_t slab = (size_t)rows * (128 * U * WK + 8) * 2, part = (size_t)WK * WN * MF * NF * 1024;
  const dim3 grid((unsigned)((p.N + 16 * NF * WN - 1) / (16 * NF * WN)), (unsigned)((p.M + 16 * MF - 1) / (16 * MF)));
  hipLaunchKernelGGL((mx_half_rows_kernel<R, MF, NF, U, WK, WN>), grid, dim3(WK * WN * 64), std::max(slab, part), s, p, rows);
}

// With 8192 columns and more, one block of columns to a workgroup gives every CU several workgroups: wider ones
// read A less often, and little per wave suffices. Below that the loads in flight per wave count. Measured, us, wide
// against narrow form: 4-bit A, 4096 -> 11008, 16 rows 12.7 / 14.4, 32 rows 14.7 / 17.8, 64 rows 19.7 / 24.8; 8 rows
// 4096 -> 4096 11.8 / 6.1, 40 rows 1000 -> 1000 7.5 / 4.8. fp16 A, 1 row 4096 -> 11008 9.2 / 10.6, 11008 -> 4096
// 11.0 / 9.6; 16 rows 4096 -> 11008 13.3 / 21.3, 8192 -> 1024 15.5 / 10.7; 64 rows 4096 -> 11008 26.6 / 39.4,
// 4096 -> 4096 25.5 / 19.8. Next to the border (weights in the Infinity Cache): 4096 -> 6144, 64 rows 4-bit A 18.7 / 17.0, fp16 A
// 24.0 / 18.4; 4096 -> 8192 19.0 / 17.3 and 25.6 / 20.7, 8 rows 11.6 / 8.6 and 10.4 / 8.7, but 1024 -> 8192 in fp16, 8 rows 4.2 / 6.0;
// 4096 -> 16384, 64 rows 19.4 / 31.5 and 26.9 / 39.1. For 8192 columns themselves the narrow forms are the faster ones with much K.
void launch_rows(bool fp4, const MxParams &p, hipStream_t s) {
  const bool wide = p.N >= 8192;
  if (fp4) {
    if (p.M <= 4 || (p.M <= 16 && !wide))
      launch_fp4_rows<1, 1, 4>(p, s);
    else if (p.M <= 16)
      launch_fp4_rows<1, 4, 2>(p, s);
    else if (!wide)
      launch_fp4_rows<2, 2, 2>(p, s);
    else if (p.M <= 32)
      launch_fp4_rows<2, 4, 2>(p, s);
    else
      launch_fp4_rows<4, 4, 1>(p, s);
  } else if (p.M <= 4) {
    if (wide)
      launch_half_rows<4, 1, 1, 1, 8, 1>(p, s);
    else
      launch_half_rows<4, 1, 1, 2, 8, 1>(p, s);
  } else if (p.M <= 16) {
    if (wide)
      launch_half_rows<16, 1, 1, 1, 4, 2>(p, s);
    else
      launch_half_rows<16, 1, 1, 2, 8, 1>(p, s);
  } else if (p.M <= 32) {
    launch_half_rows<32, 2, 1, 1, 4, 2>(p, s);
  } else if (wide) {
    launch_half_rows<64, 4, 2, 1, 4, 2>(p, s);
  } else {
    launch_half_rows<64, 4, 1, 1, 4, 2>(p, s);
  }
}

}  // namespace

int check_mxfp4_gemm(const MxGemmDesc &d, CError *err) {
  if (d.a_dtype != GN_F16 && d.a_dtype != GN_MXFP4)
    return set_error(err, -1, "mxfp4 gemm: unsupported dtype %d of A", d.a_dtype);
  size_t n;
  if (d.K > kMaxK) return set_error(err, -1, "mxfp4 gemm: K of %ld is too large", d.K);
  if (d.M < 0 || d.N < 0 || d.K < 0) return set_error(err, -1, "mxfp4 gemm: negative size");
  // A launch has below 2^32 work-items; up to 512 of them take 16 columns, 256 take 64 rows.
  if (d.M > kMaxRows || d.N > kMaxRows) return set_error(err, -1, "mxfp4 gemm: %ld x %ld is too large", d.M, d.N);
  if (!act_supported(d.act)) return set_error(err, -1, "mxfp4 gemm: unsupported activation %d", d.act);
  if (d.M == 0 || d.N == 0) return 0;
  if (!d.C) return set_error(err, -1, "mxfp4 gemm: NULL C");
  if (d.ldc < d.N) return set_error(err, -1, "mxfp4 gemm: leading dimension smaller than row length");
  if ((uintptr_t)d.C % 4 || (uintptr_t)d.bias % 4) return set_error(err, -1, "mxfp4 gemm: C or bias not aligned to fp32");
  if (!matrix_bytes(d.M, d.ldc, 4, &n) || n > ((size_t)1 << 62) || (d.M + 15) / 16 > (1L << 26) / ((d.N + 15) / 16))
    return set_error(err, -1, "mxfp4 gemm: problem too large for the grid");
  if (d.K == 0) return 0;
  if (int rc = check_mxfp4_matrix("mxfp4 gemm: B", d.B, d.b_scales, d.N, d.K, err)) return rc;
  if (d.a_dtype == GN_MXFP4) return check_mxfp4_matrix("mxfp4 gemm: A", d.A, d.a_scales, d.M, d.K, err);
  if (d.a_scales) return set_error(err, -1, "mxfp4 gemm: scales given for an fp16 A");
  if (d.lda > kMaxK && d.M > 1) return set_error(err, -1, "mxfp4 gemm: leading dimension %ld of A is too large", d.lda);
  return check_plain_matrix("mxfp4 gemm: A", GN_F16, d.A, d.M, d.K, d.lda, err);
}

int launch_mxfp4_gemm(const MxGemmDesc &d, hipStream_t s, CError *err) {
  if (d.M == 0 || d.N == 0) return 0;
  MxParams p{};
  p.A = d.A;
  p.as = static_cast<const uint8_t *>(d.a_scales);
  p.B = d.B;
  p.bs = static_cast<const uint8_t *>(d.b_scales);
  p.G = (int)groups_of(d.K);
  p.C = d.C;
  p.bias = d.bias;
  p.M = d.M, p.N = d.N, p.K = d.K, p.lda = d.lda, p.ldc = d.ldc;
  p.alpha = d.alpha, p.beta = d.beta, p.act = d.act, p.act_alpha = d.act_alpha;
  if (d.K == 0) {
    hipLaunchKernelGGL(mx_k0_kernel, dim3(grid_of(d.M * d.N, 256)), dim3(256), 0, s, p);
  } else {
    // The few-rows kernels against tiles, us, weights in the Infinity Cache. fp16 A: 4096 -> 4096, 16 rows 7.7 / 18.1, 64 rows
    // 18.2 / 18.6; 11008 -> 4096, 64 rows 43.8 / 42.7; 4096 -> 11008, 32 rows 16.7 / 18.4, 64 rows 25.9 / 19.2. 4-bit A: 4096 -> 4096, 16
    // rows 6.4 / 8.1, 64 rows 10.1 / 8.6; 11008 -> 4096, 64 rows 15.9 / 17.3; 4096 -> 11008, 1 row 8.7 / 8.1, 64 rows 19.1 / 8.8. The border
    // fits where a tile to a CU does not go round; with many columns tiles would win below it, in 4 bits at any number of rows.
    if (d.M <= 64)
      launch_rows(d.a_dtype == GN_MXFP4, p, s);
    else if (d.a_dtype == GN_MXFP4)
      launch_fp4_tiles(p, s);
    else
      launch_half_tiles(p, s);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : hip_error(err, -6, "mxfp4 gemm launch", e);
}

}  // namespace gn
