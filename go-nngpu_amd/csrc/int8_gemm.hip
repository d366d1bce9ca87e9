// int8_gemm.hip — products of 8-bit integers, C = act(alpha (sum_k A B) b_scale a_scale + beta C + bias).
//
// The sums are exact in 32 bits (K below 2^17). A sum becomes fp32, is multiplied by its column's scale, and then by alpha times its
// row's in one step with the addition of what beta and the bias give.
//
// Times in this file: of a kernel among others in a captured graph, on three sets of inputs in turn, so that weights of up to some 80 MB
// come from the Infinity Cache. They differ by 2 to 5% from run to run.
#include <algorithm>
#include <climits>

#include "gemm_tile.h"
#include "int8.h"
#include "int8_round.h"

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

// Offset v of a copy that begins at k if that is below left, else one out of range. (Without a comparison, whose result
// would take scalar registers for each of a wave's copies.)
__device__ __forceinline__ unsigned below(unsigned v, int k, int left) { return v | ((unsigned)(left - 1 - k) & kOutOfRange); }

// The first `n` bytes of v, zeros after them.
__device__ __forceinline__ i32x4_t first_bytes(i32x4_t v, int n) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int left = n - 4 * i;
    v[i] = left >= 4 ? v[i] : left <= 0 ? 0 : v[i] & ((1 << (8 * left)) - 1);
  }
  return v;
}

struct __attribute__((packed, aligned(4))) Unaligned4 {
  float4_t v;  // the hardware takes vectors at any address that is a multiple of 4
};

// The factor of a row's sums, and what becomes of a sum times its column's scale.
__device__ __forceinline__ float row_factor(const Int8Params &p, long m) { return p.as ? p.alpha * p.as[m] : p.alpha; }
__device__ __forceinline__ float finish(const Int8Params &p, float v, float factor, long m, long n) {
  float t = p.bias ? p.bias[n] : 0.0f;
  if (p.beta != 0.0f) t = fmaf(p.beta, p.C[m * p.ldc + n], t);
  return apply_act(p.act, fmaf(v, factor, t), p.act_alpha);
}
// Columns n .. n + 3 of row m, those inside the matrix.
__device__ __forceinline__ void finish4(const Int8Params &p, i32x4_t q, float factor, long m, long n) {
  if (n + 3 < p.N) {
    const float4_t one = {1.0f, 1.0f, 1.0f, 1.0f}, zero = {0.0f, 0.0f, 0.0f, 0.0f};
    const float4_t b = p.bs ? reinterpret_cast<const Unaligned4 *>(p.bs + n)->v : one;
    float4_t v = p.bias ? reinterpret_cast<const Unaligned4 *>(p.bias + n)->v : zero;
    float *dst = p.C + m * p.ldc + n;
    if (p.beta != 0.0f) {
      const float4_t old = reinterpret_cast<const Unaligned4 *>(dst)->v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = fmaf(p.beta, old[e], v[e]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = apply_act(p.act, fmaf((float)q[e] * b[e], factor, v[e]), p.act_alpha);
    reinterpret_cast<Unaligned4 *>(dst)->v = v;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < p.N) p.C[m * p.ldc + n + e] = finish(p, (float)q[e] * (p.bs ? p.bs[n + e] : 1.0f), factor, m, n + e);
  }
}

// K == 0: act(beta C + bias).
__global__ void __launch_bounds__(256) i8_k0_kernel(Int8Params p) {
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < p.M * p.N; i += (long)gridDim.x * 256)
    p.C[i / p.N * p.ldc + i % p.N] = finish(p, 0.0f, 1.0f, i / p.N, i % p.N);
}

// ------------------------------------------------------------------ small products
// A workgroup takes 16 MF rows and 16 NF columns; its KW waves cut K among them, in steps of S bytes that they take in turn, and
// their sums meet in LDS at the end. Each wave copies what it multiplies into slots of its own, NS steps ahead, so nothing is
// waited for but a wave's own copies: there is no barrier in the loop.
// A fragment asked for from memory as the instruction wants it (lane % 16 its row) spreads each four lanes over four rows, which a
// CU's address unit takes at 38 KB/us, from the caches too; copied to LDS in whole pieces of S bytes to a row the same
// bytes come at up to 90 (from L2; the Infinity Cache gives all CUs together 7.5 TB/s, 29 KB/us each).
// A chunk of 1 KiB is RPC rows of S bytes; octet o of a row sits at place o ^ swizzle(row): the 16 rows that a phase of a fragment
// read touches fall on distinct banks.
// What bounds them is a chain of latencies: 27 rows 2027 -> 4099 in 5.2 us and 64 rows 4096 -> 4096 in 7.5, the waves waiting for 45% of their
// cycles.
template <int S>
struct Chunk {
  static_assert(S == 64 || S == 128, "bytes to a row");
  static constexpr int RPC = 1024 / S, OCTETS = S / 16;
  static __device__ __forceinline__ int swizzle(int row) { return S == 128 ? (row >> 1) & 7 : (row >> 2) & 3; }
  static __device__ __forceinline__ int row(int lane) { return lane / OCTETS; }                            // of the chunk
  static __device__ __forceinline__ int octet(int row, int lane) { return (lane % OCTETS) ^ swizzle(row); }
  static __device__ __forceinline__ unsigned place(int row, int o) { return row * S + 16 * (o ^ swizzle(row)); }
};

// dma16 from voff + soff; both together below 2^31 where voff is in range.
__device__ __forceinline__ void dma16_at(const BufRsrc &s, unsigned voff, unsigned soff, unsigned lds) {
  int saved;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %4\n\t"
      "buffer_load_dwordx4 %1, %2, %3 offen lds\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(saved)
      : "v"(voff), "s"(s.r), "s"(soff), "s"(lds)
      : "memory");
}

// The waves' sums of MF x NF blocks, which take the slots' place in LDS, added up: write(i, j, v) for each block, by one wave.
template <int MF, int NF, int KW, typename F>
__device__ __forceinline__ void join_waves(char *smem, const i32x4_t (&acc)[MF][NF], int wave, int lane, F write) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();  // no copy is under way
  i32x4_t *part = reinterpret_cast<i32x4_t *>(smem);
  if (wave < KW) {  // there may be others
#pragma unroll
    for (int i = 0; i < MF; ++i)
#pragma unroll
      for (int j = 0; j < NF; ++j) part[(wave * MF * NF + i * NF + j) * 64 + lane] = acc[i][j];
  }
  __syncthreads();
#pragma unroll 1
  for (int f = wave; f < MF * NF; f += blockDim.x / 64) {
    i32x4_t v = part[f * 64 + lane];
#pragma unroll
    for (int w = 1; w < KW; ++w) v += part[(w * MF * NF + f) * 64 + lane];
    write(f / NF, f % NF, v);
  }
}

template <int MF, int NF, int KW, int S, int NS>
__global__ void __launch_bounds__(KW * 64) i8_stream_kernel(Int8Params p) {
  using C = Chunk<S>;
  constexpr int H = S / 64;                                // instructions' k to a step
  constexpr int CA = 16 * MF / C::RPC, CB = 16 * NF / C::RPC, CPS = CA + CB, SLOT = CPS * 1024;
  constexpr int RING = KW * NS * SLOT, PART = KW * MF * NF * 1024;
  static_assert(CA >= 1 && CB >= 1 && (NS - 1) * CPS < 64, "copies");
  __shared__ __attribute__((aligned(1024))) char smem[RING > PART ? RING : PART];
  int tm, tn;
  tile_coords(p, tm, tn);
  const long m0 = (long)tm * 16 * MF, n0 = (long)tn * 16 * NF;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;

  const BufRsrc da = make_rsrc(static_cast<const char *>(p.A) + m0 * p.lda), db = make_rsrc(static_cast<const char *>(p.B) + n0 * p.ldb);
  unsigned va[CA], vb[CB];
  int ka[CA], kb[CB];
#pragma unroll
  for (int i = 0; i < CA; ++i) {
    const int row = C::RPC * i + C::row(lane);
    ka[i] = 16 * C::octet(row, lane);
    va[i] = m0 + row < p.M ? (unsigned)(row * p.lda) + ka[i] : kOutOfRange;
  }
#pragma unroll
  for (int i = 0; i < CB; ++i) {
    const int row = C::RPC * i + C::row(lane);
    kb[i] = 16 * C::octet(row, lane);
    vb[i] = n0 + row < p.N ? (unsigned)(row * p.ldb) + kb[i] : kOutOfRange;
  }
  const unsigned lds = lds_offset(smem) + wave * NS * SLOT;
  const int K = (int)p.K;
  auto issue = [&](int t, int slot) {  // of the wave's steps; past K all reads are zeros
    const int k = (wave + t * KW) * S, left = K - k;
    const unsigned to = lds + slot * SLOT;
    if (left >= S) {
#pragma unroll
      for (int i = 0; i < CB; ++i) dma16_at(db, vb[i], k, __builtin_amdgcn_readfirstlane(to + (CA + i) * 1024));
#pragma unroll
      for (int i = 0; i < CA; ++i) dma16_at(da, va[i], k, __builtin_amdgcn_readfirstlane(to + i * 1024));
    } else {
#pragma unroll
      for (int i = 0; i < CB; ++i)
        dma16_at(db, below(vb[i], kb[i], left), left > 0 ? k : 0, __builtin_amdgcn_readfirstlane(to + (CA + i) * 1024));
#pragma unroll
      for (int i = 0; i < CA; ++i)
        dma16_at(da, below(va[i], ka[i], left), left > 0 ? k : 0, __builtin_amdgcn_readfirstlane(to + i * 1024));
    }
  };
  i32x4_t acc[MF][NF];
#pragma unroll
  for (int i = 0; i < MF; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) acc[i][j] = i32x4_t{0, 0, 0, 0};
  const int steps = (K + S - 1) / S, mine = wave < steps ? (steps - wave + KW - 1) / KW : 0;
#pragma unroll 1
  for (int t = 0; t < NS; ++t) issue(t, t);
  int slot = 0;
  for (int t = 0; t < mine; ++t) {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NS - 1) * CPS) : "memory");
    const char *at = smem + (wave * NS + slot) * SLOT;
    i32x4_t a[H][MF], b[H][NF];
#pragma unroll
    for (int h = 0; h < H; ++h) {
#pragma unroll
      for (int j = 0; j < NF; ++j) b[h][j] = *reinterpret_cast<const i32x4_t *>(at + CA * 1024 + C::place(16 * j + r, 4 * h + g));
#pragma unroll
      for (int i = 0; i < MF; ++i) a[h][i] = *reinterpret_cast<const i32x4_t *>(at + C::place(16 * i + r, 4 * h + g));
    }
    const int left = K - (wave + t * KW) * S;
    if (left < S) {  // A's bytes past K, which belong to its rows, as zeros
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int i = 0; i < MF; ++i) a[h][i] = first_bytes(a[h][i], left - 64 * h - 16 * g);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the slot has been read
    issue(t + NS, slot);
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int j = 0; j < NF; ++j) acc[i][j] = mfma_i8(b[h][j], a[h][i], acc[i][j]);
    slot = slot + 1 == NS ? 0 : slot + 1;
  }
  join_waves<MF, NF, KW>(smem, acc, wave, lane, [&](int i, int j, i32x4_t v) {
    const long m = m0 + 16 * i + r;
    if (m < p.M) finish4(p, v, row_factor(p, m), m, n0 + 16 * j + 4 * g);
  });
}

// Up to kMaxTokens rows of activations that the kernel brings to 8 bits itself, into LDS: a launch and a wait for it less than with a
// kernel before it. QW waves do that while the first weights of the KW others are on their way (a wave's own wait for the rows would be
// one for its weights too). One row 4096 -> 11008 takes 11.5 us (14.5 with weights from memory), of which its 45 MB would take 8.8 at a large
// copy's rate: one workgroup to a CU, whose start, first weights and join nothing overlaps. 11008 -> 4096 takes 12.8 (16.4) and 4096 -> 4096
// 6.9 (7.9; 3.3 at that rate): with 16 columns to a workgroup 32 KiB of a CU's 64 or 172 are on their way while the row is quantised.
constexpr int kMaxTokens = 4;
__host__ __device__ inline int token_pitch(long K) { return (int)((K + 127) / 128 * 128 + 16); }  // rows on distinct banks
template <typename T, int NF, int KW, int NS, int QW>
__global__ void __launch_bounds__((KW + QW) * 64) i8_token_kernel(Int8Params p, const T *x, long ldx, const float *col_scale) {
  using C = Chunk<128>;
  constexpr int CB = 16 * NF / C::RPC, SLOT = CB * 1024;
  constexpr int RING = KW * NS * SLOT, PART = KW * NF * 1024;
  static_assert((NS - 1) * CB < 64 && RING >= PART, "copies");
  static_assert(QW % kMaxTokens == 0 && kMaxTokens == 4, "waves to a row");
  __shared__ uint32_t tops[QW];
  __shared__ float scales[kMaxTokens];
  extern __shared__ __attribute__((aligned(1024))) char smem[];  // the slots, in the end the partial sums; the rows in 8 bits
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int M = (int)p.M, K = (int)p.K, pitch = token_pitch(K), end = pitch - 16;
  char *rows = smem + RING;
  const int per = M == 1 ? QW : M == 2 ? QW / 2 : QW / kMaxTokens;  // waves to a row

  unsigned vb[CB];
  int kb[CB];
  const BufRsrc db = make_rsrc(static_cast<const char *>(p.B) + (long)blockIdx.x * 16 * NF * p.ldb);
#pragma unroll
  for (int i = 0; i < CB; ++i) {
    const int br = C::RPC * i + C::row(lane);
    kb[i] = 16 * C::octet(br, lane);
    vb[i] = (long)blockIdx.x * 16 * NF + br < p.N ? (unsigned)(br * p.ldb) + kb[i] : kOutOfRange;
  }
  const unsigned lds = lds_offset(smem) + wave * NS * SLOT;
  auto issue = [&](int t, int slot) {  // of the wave's steps; past K all reads are zeros
    const int k = (wave + t * KW) * 128, left = K - k;
    const unsigned to = lds + slot * SLOT;
    if (left >= 128) {
#pragma unroll
      for (int i = 0; i < CB; ++i) dma16_at(db, vb[i], k, __builtin_amdgcn_readfirstlane(to + i * 1024));
    } else {
#pragma unroll
      for (int i = 0; i < CB; ++i)
        dma16_at(db, below(vb[i], kb[i], left), left > 0 ? k : 0, __builtin_amdgcn_readfirstlane(to + i * 1024));
    }
  };
  const int part = (wave - KW) % per, first = (wave - KW) / per;
  // The values from `at` on times their columns' factors, zeros past the row.
  auto load = [&](int m, int at, float (&y)[8]) {
    Eight<T> v;
    v.load(x + m * ldx + at, K - at);
    if (col_scale) {
      Eight<float> c;
      c.load(col_scale + at, K - at);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = v[i] * c[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = v[i];
    }
  };
  auto top_of = [&](int m) {
    uint32_t top = 0;
#pragma unroll 1
    for (int at = 8 * (part * 64 + lane); at < K; at += 8 * per * 64) {
      float y[8];
      load(m, at, y);
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(y[i]) & 0x7fffffffu);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
    return top;
  };
  auto quantize = [&](int m, uint32_t top) {
    const float s = int8_scale(top), inv = 1.0f / s;
    if (part == 0 && lane == 0) scales[m] = s;
#pragma unroll 1
    for (int at = 8 * (part * 64 + lane); at < end; at += 8 * per * 64) {  // zeros from K on
      float y[8];
      load(m, at, y);
      *reinterpret_cast<u32x2_t *>(rows + m * pitch + at) = int8_round8(y, s, inv);
    }
  };
  if (wave < KW) {
#pragma unroll 1
    for (int t = 0; t < NS; ++t) issue(t, t);
    lds_barrier();
  } else {
    uint32_t top = first < M ? top_of(first) : 0;
    if (lane == 0) tops[wave - KW] = top;
    lds_barrier();
    if (first < M) {
      for (int w = 0; w < per; ++w) top = max(top, tops[first * per + w]);
      quantize(first, top);
    }
  }
  lds_barrier();

  i32x4_t acc[1][NF];
#pragma unroll
  for (int j = 0; j < NF; ++j) acc[0][j] = i32x4_t{0, 0, 0, 0};
  const int steps = (K + 127) / 128, count = wave < min(steps, KW) ? (steps - wave + KW - 1) / KW : 0;
  const char *arow = rows + min(r, M - 1) * pitch + 16 * g;
  int slot = 0;
  for (int t = 0; t < count; ++t) {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NS - 1) * CB) : "memory");
    const char *at = smem + (wave * NS + slot) * SLOT;
    i32x4_t a[2], b[2][NF];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int j = 0; j < NF; ++j) b[h][j] = *reinterpret_cast<const i32x4_t *>(at + C::place(16 * j + r, 4 * h + g));
      a[h] = *reinterpret_cast<const i32x4_t *>(arow + (wave + t * KW) * 128 + 64 * h);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the slot has been read
    issue(t + NS, slot);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < NF; ++j) acc[0][j] = mfma_i8(b[h][j], a[h], acc[0][j]);
    slot = slot + 1 == NS ? 0 : slot + 1;
  }
  // What only the end needs of the arguments is read again: kept through the quantisation it takes scalar registers that it has not.
  auto *args = (const CONST_AS Int8Params *)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(args));
  const Int8Params q = *(const Int8Params *)args;
  join_waves<1, NF, KW>(smem, acc, wave, lane, [&](int, int j, i32x4_t v) {
    if (r < (int)q.M) finish4(q, v, q.alpha * scales[r], r, (long)blockIdx.x * 16 * NF + 16 * j + 4 * g);
  });
}

// ------------------------------------------------------------------ many rows
// WM x WN waves, each FM x FN blocks of 16 x 16. K goes in pieces of 128 bytes to a row, copied straight to LDS by dma16 in chunks
// of 8 rows (ring_plan.h's places: a wave's copies are whole 128-byte lines, its fragment reads fall on distinct banks), HS pieces to a
// stage and NS stages in LDS. A piece is two steps of 64 k: while one is multiplied the next one's fragments are read, and before a
// stage's last the next stage has landed (one wait and one barrier to a stage). Two pieces to a stage are for tiles whose
// barrier weighs more than their products and which leave the room in LDS (512 rows 11008 -> 4096, 64 x 128 tiles: 34.6 us with one, 31.8; 256
// rows 4096 -> 4096, 64 x 64 tiles 11.9 / 10.5; with four waves, of which two workgroups share a CU, 11.5 / 11.0 and 39.5 / 45.7).
// Where K ends inside a chunk of 16 the wave that copied it clears A's bytes past K before that barrier.
// What bounds them: with 8192^3 the power that the matrix instructions take (442 us, 2.49 POP/s, at 1.7 GHz, the matrix units busy for 68% of
// the cycles), with one tile to a CU the stages' latency (512 rows 4096 -> 11008 in 30 us, 11008 -> 4096 in 33: copies, fragments and
// barriers take a piece of 128 x 192 1291 cycles, where the matrix instructions alone take 768).
template <int WM, int WN, int FM, int FN, int NS, int HS>
struct I8Tile {
  static constexpr int BM = WM * FM * 16, BN = WN * FN * 16, PIECE = (BM + BN) * 128, STAGE = HS * PIECE;
  static constexpr int ALL = BM * (BN + 4) * 4, PARTS = ALL > 140 * 1024 ? 2 : 1, SUMS = ALL / PARTS;  // the sums, all at once or in halves
  static constexpr int EPI = SUMS + (BM + 2 * BN) * 4;                                                 // with the scales and the bias
  static constexpr int BYTES = NS * STAGE > EPI ? NS * STAGE : EPI;
};
template <int WM, int WN, int FM, int FN, int NS, int HS>
__global__ void __launch_bounds__(WM * WN * 64) __attribute__((amdgpu_waves_per_eu(2, 2)))
i8_tile_kernel(Int8Params p) {
  using Tile = I8Tile<WM, WN, FM, FN, NS, HS>;
  using C = Chunk<128>;
  constexpr int NW = WM * WN, NT = NW * 64, BM = Tile::BM, BN = Tile::BN, PIECE = Tile::PIECE, STAGE = Tile::STAGE;
  constexpr int CA = BM / C::RPC / NW, CB = BN / C::RPC / NW, CPW = CA + CB;
  static_assert(CA * NW * C::RPC == BM && CB * NW * C::RPC == BN, "chunks");
  static_assert((NS - 1) * HS * CPW < 64 && (NS > 2 || (NS == 2 && HS == 1)) && FM % Tile::PARTS == 0 && NT >= BN / 4, "copies and rows");
  __shared__ __attribute__((aligned(1024))) char smem[Tile::BYTES];

  int tm, tn;
  tile_coords(p, tm, tn);
  const long m0 = (long)tm * BM, n0 = (long)tn * BN;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wm = wave / WN, wn = wave % WN, r = lane & 15, g = lane >> 4;
  const int pieces = (int)((p.K + 127) / 128), ns = (pieces + HS - 1) / HS;

  // What the epilogue needs of each row and column: the rows' scales, the columns' scales and biases, thread by thread; not
  // touched, which would be a wait for them, until the stages are done with LDS.
  constexpr int LINES = BM + 2 * BN, SPT = (LINES + NT - 1) / NT;
  float line[SPT];
#pragma unroll
  for (int i = 0; i < SPT; ++i) {
    const int at = threadIdx.x + i * NT;
    line[i] = at < BM + BN ? 1.0f : 0.0f;
    if (at < BM) {
      if (p.as && m0 + at < p.M) line[i] = p.as[m0 + at];
    } else if (at < BM + BN) {
      if (p.bs && n0 + at - BM < p.N) line[i] = p.bs[n0 + at - BM];
    } else if (at < LINES) {
      if (p.bias && n0 + at - BM - BN < p.N) line[i] = p.bias[n0 + at - BM - BN];
    }
  }

  const char *a0 = static_cast<const char *>(p.A) + m0 * p.lda, *b0 = static_cast<const char *>(p.B) + n0 * p.ldb;
  unsigned va[CA], vb[CB];
  // A copy's first k in the stage, for even i; for odd i the octet's upper bit is the other way round (row >> 1 is 4 more).
  const int ka = 16 * C::octet(C::RPC * wave * CA + C::row(lane), lane), kb = 16 * C::octet(C::RPC * wave * CB + C::row(lane), lane);
  auto k_of = [](int k, int i) { return k ^ (i & 1 ? 64 : 0); };
#pragma unroll
  for (int i = 0; i < CA; ++i) {
    const int row = C::RPC * (wave * CA + i) + C::row(lane);
    va[i] = m0 + row < p.M ? (unsigned)(row * p.lda) + k_of(ka, i) : kOutOfRange;
  }
#pragma unroll
  for (int i = 0; i < CB; ++i) {
    const int row = C::RPC * (wave * CB + i) + C::row(lane);
    vb[i] = n0 + row < p.N ? (unsigned)(row * p.ldb) + k_of(kb, i) : kOutOfRange;
  }
  const unsigned lds = lds_offset(smem);
  // Part q of `parts` of a side's copies of piece h of stage t into a slot; chunks that begin at or past K read zeros.
  auto issue = [&](const char *base, const unsigned *v, int k, int count, int t, unsigned to, int q, int parts) {
    const int left = (int)p.K - 128 * t;
    const BufRsrc d = make_rsrc(base + 128L * t);
#pragma unroll
    for (int i = 0; i < count; ++i)
      if (i * parts / count == q) dma16(d, below(v[i], k_of(k, i), left), __builtin_amdgcn_readfirstlane(to + i * 1024));
  };
  auto issue_a = [&](int t, int h, int slot, int q, int parts) {
    issue(a0, va, ka, CA, t * HS + h, lds + slot * STAGE + h * PIECE + wave * CA * 1024, q, parts);
  };
  auto issue_b = [&](int t, int h, int slot, int q, int parts) {
    issue(b0, vb, kb, CB, t * HS + h, lds + slot * STAGE + h * PIECE + BM * 128 + wave * CB * 1024, q, parts);
  };
  // This wave's chunks of A of the last piece, once they have landed (all that is under way behind them reads zeros).
  auto clear_tail = [&](int slot) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const int left = (int)p.K - 128 * (pieces - 1), h = (pieces - 1) % HS;
#pragma unroll
    for (int i = 0; i < CA; ++i) {
      const int n = left - k_of(ka, i);
      if (n > 0 && n < 16) {
        i32x4_t *c = reinterpret_cast<i32x4_t *>(smem + slot * STAGE + h * PIECE + (wave * CA + i) * 1024 + lane * 16);
        *c = first_bytes(*c, n);
      }
    }
  };

  i32x4_t fa[2][FM], fb[2][FN];
  // Of step h of a stage, which is half a piece.
  auto read_a = [&](int slot, int h, int i) {
    fa[h & 1][i] = *reinterpret_cast<const i32x4_t *>(smem + slot * STAGE + h / 2 * PIECE + C::place((wm * FM + i) * 16 + r, 4 * (h & 1) + g));
  };
  auto read_b = [&](int slot, int h, int j) {
    fb[h & 1][j] =
        *reinterpret_cast<const i32x4_t *>(smem + slot * STAGE + h / 2 * PIECE + BM * 128 + C::place((wn * FN + j) * 16 + r, 4 * (h & 1) + g));
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
      for (int j = 0; j < FN; ++j) acc[i][j] = mfma_i8(fb[h][j], fa[h][i], acc[i][j]);
  };

  const bool tail = p.K % 16 != 0;
  // With two slots the first copies are all before the loop, with more all but the first of the last stage's are in it.
  constexpr bool SPREAD = NS > 2;
#pragma unroll 1
  for (int t = 0; t < NS; ++t) {
#pragma unroll
    for (int h = 0; h < HS; ++h) {
      const bool all = !SPREAD || t < NS - 1;
      if (all || h == 0) issue_a(t, h, t, 0, 1);
      if (all) issue_b(t, h, t, 0, 1);
    }
  }
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(SPREAD ? (NS - 2) * HS * CPW + CA : (NS - 1) * HS * CPW));
  if (tail && ns == 1) clear_tail(0);
  __syncthreads();
  read_part(0, 0, 0, 1);
  int cur = 0, prev = NS - 1;
  for (int t = 0; t < ns; ++t) {
    const int nxt = cur + 1 == NS ? 0 : cur + 1;
    auto arrive = [&] {  // stage t + 1 is there, in all waves
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_waitcnt(vmcnt_imm((NS - 2) * HS * CPW));
      if (tail && t + 2 == ns) clear_tail(nxt);
      __syncthreads();
      __builtin_amdgcn_sched_barrier(0);
    };
    if constexpr (SPREAD) {
      // A step's products, row by row, with the next step's fragments and a share of the copies behind each row: a copy takes the
      // address unit 20 cycles, and a wave that meets a full one waits there with all that it has behind it. B's copies of a stage wait
      // for the step after A's. (All copies after the barrier, 512 rows 11008 -> 4096: 128 x 256 tiles 68 us instead of 57, 128 x 192 54.6 /
      // 50.5, 128 x 128 42 / 41.)
      auto step = [&](int h, int read_slot, auto copies) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < FM; ++i) {
          mfma_rows(h & 1, i, i + 1);
          read_part(read_slot, h + 1 < 2 * HS ? h + 1 : 0, i, FM);
          __builtin_amdgcn_sched_barrier(0);
          copies(i);
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      step(0, cur, [&](int i) { issue_b(t + NS - 1, 0, prev, i, FM); });
      if constexpr (HS == 2) {
        step(1, cur, [&](int i) { issue_a(t + NS - 1, 1, prev, i, FM); });
        step(2, cur, [&](int i) { issue_b(t + NS - 1, 1, prev, i, FM); });
      }
      arrive();
      step(2 * HS - 1, nxt, [&](int i) { issue_a(t + NS, 0, cur, i, FM); });
    } else {
      // Two slots leave no step to spread the copies over: in two bursts, each once the matrix instructions have work (8192^3 440 us; row
      // by row 472; four slots of half a stage, with a barrier to each, 484).
      constexpr int R0 = FM / 2, NR = FM / 2 + FN / 2;
      __builtin_amdgcn_sched_barrier(0);
      read_part(cur, 1, 0, 1);
      mfma_rows(0, 0, FM);
      sched_interleave<FM * FN, FM + FN>();
      arrive();
      mfma_rows(1, 0, 1);
      __builtin_amdgcn_sched_barrier(0);
      issue_a(t + NS, 0, cur, 0, 1);
      read_part(nxt, 0, 0, 2);
      mfma_rows(1, 1, R0);
      sched_interleave<(R0 - 1) * FN, NR>();
      __builtin_amdgcn_sched_barrier(0);
      mfma_rows(1, R0, R0 + 1);
      __builtin_amdgcn_sched_barrier(0);
      issue_b(t + NS, 0, cur, 0, 1);
      read_part(nxt, 0, 1, 2);
      mfma_rows(1, R0 + 1, FM);
      sched_interleave<(FM - R0 - 1) * FN, NR>();
    }
    prev = cur, cur = nxt;
  }
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
  __syncthreads();  // no copy is under way and all waves are done with the stages: the sums take their place
  // The sides of the products are changed, so that lane (r, g) of a block has row r, columns 4 g .. 4 g + 3: one 16-byte write to
  // LDS for each block, and from there whole rows of the tile go out through a short loop. Straight code for all of
  // a thread's sums, as the other products' epilogue has it, costs more in instructions that nobody has in a cache yet (70 KB of
  // code; a single tile of 256 x 256 with K = 128 took 13.5 us) than what it does.
  float *sa = reinterpret_cast<float *>(smem + Tile::SUMS), *sb = sa + BM, *bias = sb + BN;
#pragma unroll
  for (int i = 0; i < SPT; ++i) {
    const int at = threadIdx.x + i * NT;
    if (at < LINES) sa[at] = at < BM ? p.alpha * line[i] : line[i];
  }
  constexpr int LP = BN + 4, CPR = BN / 4, RPS = NT / CPR, PARTS = Tile::PARTS, FP = FM / PARTS, ROWS = BM / PARTS;
  int *sums = reinterpret_cast<int *>(smem);
  const int c4 = threadIdx.x % CPR, r0 = threadIdx.x / CPR;  // threads with r0 >= RPS only write to LDS
  const long col = n0 + 4 * c4;
  auto dump = [&](auto part) {
    constexpr int P = decltype(part)::value;
#pragma unroll
    for (int i = 0; i < FP; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
        *reinterpret_cast<i32x4_t *>(sums + ((wm * FP + i) * 16 + r) * LP + (wn * FN + j) * 16 + 4 * g) = acc[P * FP + i][j];
  };
  auto sweep = [&](int part, auto act_c) {
    constexpr int ACT = decltype(act_c)::value;
    const int act = ACT == kActRuntime ? p.act : ACT;
    const float4_t bs = *reinterpret_cast<const float4_t *>(sb + 4 * c4), bv = *reinterpret_cast<const float4_t *>(bias + 4 * c4);
#pragma unroll 2
    for (int t = r0; t < ROWS; t += RPS) {
      const int row = (t / (FP * 16) * FM + part * FP) * 16 + t % (FP * 16);  // of the tile
      if (m0 + row >= p.M) continue;
      const i32x4_t q = *reinterpret_cast<const i32x4_t *>(sums + t * LP + 4 * c4);
      const float as = sa[row];
      float *dst = p.C + (m0 + row) * p.ldc + col;
      float4_t v = bv;
      if (col + 3 < p.N) {
        if (p.beta != 0.0f) {
          const float4_t old = reinterpret_cast<const Unaligned4 *>(dst)->v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = fmaf(p.beta, old[e], v[e]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = apply_act(act, fmaf((float)q[e] * bs[e], as, v[e]), p.act_alpha);
        __builtin_nontemporal_store(v, &reinterpret_cast<Unaligned4 *>(dst)->v);  // C is not read again: keep L2 for A and B
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (col + e < p.N) {
            if (p.beta != 0.0f) v[e] = fmaf(p.beta, dst[e], v[e]);
            dst[e] = apply_act(act, fmaf((float)q[e] * bs[e], as, v[e]), p.act_alpha);
          }
        }
      }
    }
  };
#pragma unroll 1
  for (int part = 0; part < PARTS; ++part) {
    if (part == 0)
      dump(ActCode<0>{});
    else
      dump(ActCode<PARTS - 1>{});
    lds_barrier();
    if (r0 < RPS) {
      switch (p.act) {
        case -1: sweep(part, ActCode<-1>{}); break;
        case 0: sweep(part, ActCode<0>{}); break;
        case 7: sweep(part, ActCode<7>{}); break;
        default: sweep(part, ActCode<kActRuntime>{}); break;
      }
    }
    lds_barrier();
  }
}

unsigned grid_of(long n, long per) { return (unsigned)std::max(1L, std::min((n + per - 1) / per, 1L << 20)); }

template <int MF, int NF, int KW, int S, int NS>
void launch_stream(Int8Params p, hipStream_t s) {
  p.tiles_m = (int)((p.M + 16 * MF - 1) / (16 * MF));
  p.tiles_n = (int)((p.N + 16 * NF - 1) / (16 * NF));
  p.group_m = p.tiles_m;  // the rows' blocks of some columns side by side: those columns are read once by their XCD
  hipLaunchKernelGGL((i8_stream_kernel<MF, NF, KW, S, NS>), dim3((unsigned)(p.tiles_m * p.tiles_n)), dim3(KW * 64), 0, s, p);
}

template <int WM, int WN, int FM, int FN, int NS, int HS = 1>
void launch_tiles(Int8Params p, hipStream_t s) {
  constexpr int BM = WM * FM * 16, BN = WN * FN * 16;
  p.tiles_m = (int)((p.M + BM - 1) / BM);
  p.tiles_n = (int)((p.N + BN - 1) / BN);
  hipLaunchKernelGGL((i8_tile_kernel<WM, WN, FM, FN, NS, HS>), dim3((unsigned)(p.tiles_m * p.tiles_n)), dim3(WM * WN * 64), 0, s, p);
}

// The kind of tile with which the busiest CU's share takes the least time, the first of equals. In 10 ns: fixed, and `stage` for each
// 128 of K, for a tile alone on a CU; `next`, and `more` for each 128 of K, for each further tile of its share. Fitted to
// these kinds' times on some 25 sizes from 16 to 8192 rows and 100 to 16000 columns and K; of 26 such sizes the choice takes 0.6% more than the best
// kind of each, at most 13% (32 rows 4096 -> 11008). Measured, us, 16 x 16 / 16 x 64 / 32 x 32 / 32 x 64 / 64 x 64 (8 waves) / 64 x 64 (4) / 64 x 128
// (8) / 64 x 128 (4) / 128 x 128 / 128 x 192 / 128 x 256 / 256 x 256: 4096 -> 4096, 64 rows 11.3 / 8.0 / 7.5 / 9.3 / 9.8 / 11.1 / 12.1 / 14.5 /
// 17.8 / 22.1 / 26.4 / 40.2, 256 rows 36.1 / 25.4 / 22.3 / 16.3 / 10.3 / 11.3 / 12.2 / 14.7 / 18.2 / 23.2 / 27.5 / 44.0, 2048 rows 308 / 197 /
// 205 / 131 / 68.2 / 58.7 / 55.4 / 46.8 / 43.7 / 49.1 / 35.2 / 44.3; 512 rows 4096 -> 11008 166 / 140 / 112 / 77 / 50.6 / 43.1 / 39.9 / 35.2 / 38.3 /
// 27.9 / 29.1 / 43.6, 11008 -> 4096 190 / 103 / 90 / 73 / 42.1 / 38.8 / 32.0 / 34.5 / 41.0 / 52.0 / 62.7 / 101.
struct TileCost {
  unsigned bm, bn, fixed, stage, next, more;
};
constexpr TileCost kTiles[] = {{16, 16, 329, 4, 97, 4},        {16, 64, 423, 11, 274, 10},     {32, 32, 404, 9, 252, 9},
                               {32, 64, 369, 18, 251, 16},     {64, 64, 408, 19, 228, 19},     {64, 64, 369, 24, 132, 18},
                               {64, 128, 447, 26, 218, 37},    {64, 128, 441, 34, 194, 29},    {128, 128, 555, 41, 452, 56},
                               {128, 192, 658, 54, 779, 67},   {128, 256, 689, 68, 835, 90},   {256, 256, 1084, 119, 1645, 162}};
constexpr int kKinds = sizeof(kTiles) / sizeof(kTiles[0]);
void launch_product(const Int8Params &p, hipStream_t s) {
  // One block of rows and a stream of weights longer than the model looks ahead: small workgroups, several to a CU, so that one's end
  // falls into another's stream. Against the model's choice, us, 16 rows: 4096 -> 32768 30.2 / 34.0, 50257 42.2 / 52.5, 131072 95.7 (5.6
  // TB/s) / 121; 8192 -> 17000 36.7 / 41.9; 11008 -> 65536 134 / 163; 2600 -> 131072 77.7 / 72.3, 2048 56.6 / 50.4, 1000 38.9 / 31.5.
  if (p.M <= 16 && p.N > 64 * 256 && p.K > 3584) return launch_stream<1, 2, 4, 128, 2>(p, s);
  const unsigned stages = (unsigned)(p.K + 127) / 128, M = (unsigned)p.M, N = (unsigned)p.N;
  int best = kKinds - 1;
  uint64_t least = ~0ull;
  for (int i = 0; i < kKinds; ++i) {
    const TileCost &k = kTiles[i];
    const uint64_t tiles = (uint64_t)((M + k.bm - 1) / k.bm) * ((N + k.bn - 1) / k.bn), others = (tiles - 1) / 256;  // 256 CUs
    const uint64_t cost = k.fixed + stages * k.stage + others * (k.next + stages * k.more);
    if (cost < least && tiles <= 1 << 22) best = i, least = cost;  // below 2^32 threads; the largest tiles are never more
  }
  switch (best) {
    case 0: return launch_stream<1, 1, 4, 128, 4>(p, s);
    case 1: return launch_stream<1, 4, 8, 128, 2>(p, s);
    case 2: return launch_stream<2, 2, 8, 128, 2>(p, s);
    case 3: return launch_stream<2, 4, 8, 64, 2>(p, s);
    case 4: return launch_tiles<2, 4, 2, 1, 3, 2>(p, s);
    case 5: return launch_tiles<2, 2, 2, 2, 4>(p, s);
    case 6: return launch_tiles<2, 4, 2, 2, 3, 2>(p, s);
    case 7: return launch_tiles<2, 2, 2, 4, 3>(p, s);
    case 8: return launch_tiles<2, 4, 4, 2, 3>(p, s);
    case 9: return launch_tiles<2, 4, 4, 3, 3>(p, s);
    case 10: return launch_tiles<2, 4, 4, 4, 3>(p, s);
    default: return launch_tiles<2, 4, 8, 4, 2>(p, s);
  }
}

// Up to 4 rows of activations are brought to 8 bits in the product's kernel. Against a kernel before it, us of kernels: 1 row 1000 ->
// 1000 4.5 / 5.9, 4096 -> 4096 7.4 / 8.8, 11008 -> 4096 12.9 / 15.3, 4096 -> 11008 11.7 / 12.8; 4 rows 9.7 / 9.0 and 13.8 / 13.1, where
// the other's second launch costs a caller without a graph 3 us more. The rows stand beside up to 128 KiB of slots in LDS.
bool few_tokens(long M, long K) { return M <= kMaxTokens && M * token_pitch(K) <= 24 * 1024; }
template <typename T, int NF, int KW, int NS, int QW>
void launch_token(const Int8LinearDesc &d, const Int8Params &p, hipStream_t s) {
  const int ring = KW * NF * NS * 2048;
  hipLaunchKernelGGL((i8_token_kernel<T, NF, KW, NS, QW>), dim3((unsigned)((p.N + 16 * NF - 1) / (16 * NF))), dim3((KW + QW) * 64),
                     ring + (int)p.M * token_pitch(p.K), s, p, static_cast<const T *>(d.x), d.gemm.M > 1 ? d.ldx : 0, d.col_scale);
}
template <typename T>
void launch_tokens(const Int8LinearDesc &d, const Int8Params &p, hipStream_t s) {
  // As few columns to a workgroup as leave no CU a second one: 1 row 4096 -> 4096 7.2 us with 16, 7.6 with 32, 8.8 with 64 columns;
  // 4096 -> 8192 10.8, 11.3, 11.7; 4096 -> 11008 14.4, 12.8, 11.6. Where 64 are too few for that, small workgroups of which several share a CU, so
  // that one's end falls into another's stream: 4096 -> 14000 13.6 (64 columns 13.0), 17000 15.9 (20.1), 32768 29.0 (34.6), 131072 93 (115, 5.8
  // and 4.7 TB/s); 4 rows 4096 -> 32768 40.3 (38.1), 131072 119 (139).
  if (p.N <= 16 * 256)
    launch_token<T, 1, 8, 2, 8>(d, p, s);
  else if (p.N <= 32 * 256)
    launch_token<T, 2, 8, 2, 8>(d, p, s);
  else if (p.N <= 64 * 256)
    launch_token<T, 4, 8, 2, 8>(d, p, s);
  else
    launch_token<T, 2, 4, 2, 4>(d, p, s);
}

Int8Params params_of(const Int8GemmDesc &d) {
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
  return p;
}

int launched(const char *what, CError *err) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : hip_error(err, -6, what, e);
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
  const Int8Params p = params_of(d);
  if (d.K == 0)
    hipLaunchKernelGGL(i8_k0_kernel, dim3(grid_of(d.M * d.N, 256)), dim3(256), 0, s, p);
  else
    launch_product(p, s);
  return launched("int8 gemm launch", err);
}

size_t int8_linear_workspace(long M, long N, long K) {
  size_t n;
  if (M < 1 || N < 1 || K < 1 || K > kInt8MaxK || few_tokens(M, K) || !matrix_bytes(M, int8_pitch(K) + 4, 1, &n)) return 0;
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
  if (few_tokens(g.M, g.K)) {
    const Int8Params p = params_of(g);
    if (d.dtype == GN_F16)
      launch_tokens<_Float16>(d, p, s);
    else
      launch_tokens<float>(d, p, s);
    return launched("int8 linear launch", err);
  }
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
