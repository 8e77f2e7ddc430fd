// fp8.hip — rows of 8-bit floating point with an f32 scale for each block of 128: quantising
// (bb_quantize_fp8) and the product of two sets of rows (bb_scores_fp8), on MFMA (gfx950).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>
#include <type_traits>

#include "abi.h"

namespace bb {
namespace {

constexpr int kBlock = 128;
constexpr float kE4m3Max = 448.f;
constexpr float kTiny = 0x1p-100f;  // 448 / kTiny is finite, so every finite block has a finite inverse

inline int64_t blocks_of(int64_t x) { return (x + kBlock - 1) / kBlock; }

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Vec8 {
  typedef T type __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};

// ---- quantising ---------------------------------------------------------------------------
// 16 lanes hold the 128 columns of one row's block, 8 to a lane.  The largest magnitude is
// taken over the bit patterns of |x|, whose unsigned order is finite < infinity < NaN.

// Columns [c, c + 8) of a row of d; zeros past d.
template <typename T>
__device__ __forceinline__ void load8(const T* row, int64_t c, int64_t d, float (&x)[8]) {
  if (c + 8 <= d) {
    const typename Vec8<T>::type v = *(const typename Vec8<T>::type*)(row + c);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = (float)v[j];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = c + j < d ? (float)row[c + j] : 0.f;
  }
}
__device__ __forceinline__ uint32_t top8(const float (&x)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x[j]) & 0x7FFFFFFFu;
    m = b > m ? b : m;
  }
  return m;
}
// the largest over each group of 16 lanes, to all of them
__device__ __forceinline__ uint32_t max16(uint32_t m) {
#pragma unroll
  for (int s = 1; s < 16; s *= 2) {
    const uint32_t o = (uint32_t)__shfl_xor((int)m, s, 64);
    m = o > m ? o : m;
  }
  return m;
}
// A block's scale, and what its elements are multiplied by.  Both quotients are whole f32
// divisions: the codes are defined through the rounded inverse.
__device__ __forceinline__ void block_scale(uint32_t top, float& scale, float& inv) {
  const bool finite = top < 0x7F800000u;
  const float a = fmaxf(__builtin_bit_cast(float, top), kTiny);
  scale = finite ? a / kE4m3Max : __builtin_nanf("");
  inv = finite ? kE4m3Max / a : 0.f;
}
// |x * inv| <= 448 (1 + 2^-23), which rounds to 448: no code overflows
__device__ __forceinline__ u32x2 codes8(const float (&x)[8], float inv) {
  float y[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) y[j] = inv != 0.f ? x[j] * inv : 0.f;  // (a block with an infinity or NaN: codes 0)
  u32x2 c;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h], y[4 * h + 1], 0, false);
    c[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h + 2], y[4 * h + 3], w, true);
  }
  return c;
}

struct QuantArgs {
  const void* x;
  int64_t ldx, n, d;
  uint8_t* codes;
  int64_t ld;
  float* scales;
  int64_t scales_ld;
  int32_t kb;      // blocks of a row
};

// One scale for each block of a row.  A workgroup takes one block column of 32 rows, so that
// their scales (consecutive in memory) go out as one 128-byte line.  Bound by reading the rows once and
// writing a quarter or half of that: 125,000 x 768 f32 83.7 us, 5.8 TB/s (a large copy reaches 4.7, a fill 6.8).
constexpr int kQRows = 32;
template <typename T>
__global__ __launch_bounds__(kQRows * 16) void quantize_rows_kernel(QuantArgs a) {
  const int64_t row = (int64_t)(blockIdx.x / a.kb) * kQRows + (threadIdx.x >> 4);
  const int b = blockIdx.x % a.kb;
  if (row >= a.n) return;
  const int64_t c = (int64_t)b * kBlock + (threadIdx.x & 15) * 8;
  float x[8];
  load8((const T*)a.x + row * a.ldx, c, a.d, x);
  float scale, inv;
  block_scale(max16(top8(x)), scale, inv);
  *(u32x2*)(a.codes + row * a.ld + c) = codes8(x, inv);
  if ((threadIdx.x & 15) == 0) a.scales[b * a.scales_ld + row] = scale;
}

// One scale for each 128 x 128 tile: a workgroup holds the tile in registers, so that it is read once.
// 8,192 x 4,096 bf16 18.6 us, 5.4 TB/s.
template <typename T>
__global__ __launch_bounds__(512) void quantize_tiles_kernel(QuantArgs a) {
  __shared__ uint32_t top[8];
  const int64_t r0 = (int64_t)(blockIdx.x / a.kb) * kBlock;
  const int b = blockIdx.x % a.kb;
  const int64_t c = (int64_t)b * kBlock + (threadIdx.x & 15) * 8;
  float x[4][8];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = r0 + i * 32 + (threadIdx.x >> 4);
    load8((const T*)a.x + row * a.ldx, c, row < a.n ? a.d : 0, x[i]);
    const uint32_t t = top8(x[i]);
    m = t > m ? t : m;
  }
  m = max16(m);
#pragma unroll
  for (int s = 16; s < 64; s *= 2) {
    const uint32_t o = (uint32_t)__shfl_xor((int)m, s, 64);
    m = o > m ? o : m;
  }
  if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) m = top[w] > m ? top[w] : m;
  float scale, inv;
  block_scale(m, scale, inv);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = r0 + i * 32 + (threadIdx.x >> 4);
    if (row < a.n) *(u32x2*)(a.codes + row * a.ld + c) = codes8(x[i], inv);
  }
  if (threadIdx.x == 0) a.scales[b * a.scales_ld + r0 / kBlock] = scale;
}

// ---- the product --------------------------------------------------------------------------
struct ProductArgs {
  const uint8_t *q, *x;        // codes of the queries and of the items
  const float *qs, *xs;        // their scales, [kb][...]
  int64_t ldq, ldx, ldqs, ldxs;
  void* out;
  int64_t ldo;
  int64_t M, N;
  int32_t kb;
  int32_t tile;                // the items' scales are per 128 rows
};

// One 16 x 16 product of a whole block of 128.  Lane l holds 32 bytes of row l & 15 of each operand;
// which 32 of the row's 128 is free as long as both operands agree.  Result j of lane l is row
// 4 (l >> 4) + j of the first operand against row l & 15 of the second.
//
// Two ways, chosen by the type of the scores:
//  - bf16 scores: v_mfma_f32_16x16x128_f8f6f4 on the codes as they are.  It cuts each product of a group of 8
//    (8 consecutive bytes of a lane) at 2^-13 of the group's largest before it sums them in f32 (measured:
//    the instruction's rounding is not documented; every 8-bit form does the same), an error of 1.4e-5 of the result
//    on normal inputs and at most 8 * 2^-13 = 2^-10 of the sum of magnitudes: a quarter of bf16's own half step 2^-8.
//  - f32 and f16 scores, whose half steps 2^-24 and 2^-11 are finer than that bound: the codes widened to f16, which
//    holds every e4m3 value, and v_mfma_f32_16x16x32_f16, which keeps 24 bits under the largest product (2.9e-9 on
//    the same inputs), at half the rate.
struct Narrow {
  typedef i32x8 Frag;
  static __device__ __forceinline__ Frag make(u32x4 lo, u32x4 hi) {
    return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
  }
  static __device__ __forceinline__ f32x4 dot(const Frag& a, const Frag& b) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
  }
};
struct Wide {
  struct Frag {
    f16x8 v[4];
  };
  static __device__ __forceinline__ f16x8 widen(uint32_t lo, uint32_t hi) {
    const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false);
    const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true);
    const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false);
    const f16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true);
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  }
  static __device__ __forceinline__ Frag make(u32x4 lo, u32x4 hi) {
    return Frag{{widen(lo[0], lo[1]), widen(lo[2], lo[3]), widen(hi[0], hi[1]), widen(hi[2], hi[3])}};
  }
  static __device__ __forceinline__ f32x4 dot(const Frag& a, const Frag& b) {
    f32x4 c{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.v[i], b.v[i], c, 0, 0, 0);
    return c;
  }
};
template <typename T>
using Mode = std::conditional_t<std::is_same_v<T, __bf16>, Narrow, Wide>;

// ---- the product of few rows -----------------------------------------------------------------
// Bound by reading the items once: operands go straight from memory to registers, up to PF blocks
// of a wave in flight.  A workgroup takes 16 items x 16 queries; its KS waves take every KS-th block of the
// same rows and are summed through LDS, in order of the wave.  1 x 25,216 x 384 to f32: 3.9 us, of which the launch
// is 2; 1 x 100,000 x 768: 15.5 us, 5.0 TB/s.
template <typename T, int KS, int PF>
__global__ __launch_bounds__(KS * 64) void product_few_kernel(ProductArgs a, int n_groups) {
  typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int64_t n0 = (int64_t)(blockIdx.x % n_groups) * 16, m0 = (int64_t)(blockIdx.x / n_groups) * 16;
  const bool whole = n0 + 16 <= a.N;
  // rows past the end repeat the last one: their results are not stored
  const int64_t nr = n0 + r < a.N ? n0 + r : a.N - 1, mr = m0 + r < a.M ? m0 + r : a.M - 1;
  const int64_t n = n0 + g * 4, m = m0 + r;  // this lane's scores: items n .. n + 3 of query m
  const uint8_t* xp = a.x + nr * a.ldx + g * 32;
  const uint8_t* qp = a.q + mr * a.ldq + g * 32;
  const float* xs = a.xs + (a.tile ? n0 / kBlock : n < a.N ? n : a.N - 1);
  const float* qs = a.qs + mr;
  f32x4 acc{0.f, 0.f, 0.f, 0.f};
  for (int b0 = wave; b0 < a.kb; b0 += KS * PF) {
    u32x4 x[PF][2], q[PF][2];
    f32x4 sx[PF];
    float sq[PF];
#pragma unroll
    for (int f = 0; f < PF; ++f) {
      const int b = b0 + f * KS < a.kb ? b0 + f * KS : b0;  // (a block past the end is not used below)
      const u32x4* px = (const u32x4*)(xp + (int64_t)b * kBlock);
      const u32x4* pq = (const u32x4*)(qp + (int64_t)b * kBlock);
      const float* s = xs + b * a.ldxs;
      x[f][0] = px[0];
      x[f][1] = px[1];
      q[f][0] = pq[0];
      q[f][1] = pq[1];
      sq[f] = qs[b * a.ldqs];
      if (a.tile) {
        sx[f] = f32x4{*s, *s, *s, *s};
      } else if (whole) {
        sx[f] = *(const f32x4u*)s;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) sx[f][j] = n + j < a.N ? s[j] : 0.f;
      }
    }
#pragma unroll
    for (int f = 0; f < PF; ++f) {
      if (b0 + f * KS >= a.kb) break;
      const f32x4 p = Mode<T>::dot(Mode<T>::make(x[f][0], x[f][1]), Mode<T>::make(q[f][0], q[f][1]));
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] = fmaf(sq[f] * sx[f][j], p[j], acc[j]);
    }
  }
  if constexpr (KS > 1) {
    __shared__ f32x4 part[KS - 1][64];
    if (wave > 0) part[wave - 1][lane] = acc;
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 0; w < KS - 1; ++w) acc += part[w][lane];
  }
  if (m >= a.M) return;
  typedef T Out __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  T* p = (T*)a.out + m * a.ldo + n;
  if (n + 4 <= a.N) {
    *(Out*)p = Out{(T)acc[0], (T)acc[1], (T)acc[2], (T)acc[3]};
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (n + j < a.N) p[j] = (T)acc[j];
  }
}

// ---- the product of many rows: tiles staged through LDS ----------------------------------------
// A group of WN x WM waves computes 64 WN items x 16 MT WM queries; a wave 64 items x 16 MT queries.  A
// workgroup is KG such groups, which share out the blocks of the same rows and are summed at the end.  Both
// operands' blocks of 128 codes go to LDS by LDS-DMA into D stages: the next block's loads are in flight
// while this one's products run, one barrier to a block.  The block's scales go along (4 bytes a row).
//
// LDS rows are 128 bytes of 8 chunks; chunk c of row r sits at position c ^ f(r), with f such that the 8
// rows that 8 neighbouring lanes read together have 8 different f: their 16-byte reads then fall
// on all banks once.  A lane takes chunks g and g + 4 of its row (g = lane >> 4).
//
// Item rows are dealt to MFMA tiles so that a lane's results of V neighbouring tiles are 4 V
// consecutive items: 16-byte stores, 64 bytes of a score row to each 4 lanes.
template <typename T, int WN, int WM, int MT, int D, int KG>
struct TileShape {
  static constexpr int kWaves = WN * WM, kThreads = KG * kWaves * 64;  // waves of a group, threads of all
  static constexpr int V = 4 / (int)sizeof(T);
  static constexpr int TN = WN * 64, TM = WM * MT * 16;
  static constexpr int kX = TN * kBlock, kQ = TM * kBlock, kS = (TN + TM) * 4;
  static constexpr int kStage = kX + kQ + kS;
  static constexpr int kXP = TN / 8 / kWaves, kQP = TM / 8 / kWaves;  // 1-KiB pieces of a wave
  static_assert(TN % (8 * kWaves) == 0 && TM % (8 * kWaves) == 0, "whole pieces for every wave");
  static constexpr int kSP = ((TN + TM) / 64 + kWaves - 1) / kWaves;   // 64-scale pieces of a wave
  static constexpr int kLoads = kXP + kQP + kSP;                       // loads of a wave and stage
  static_assert(TN % 64 == 0 && TM % 64 == 0, "whole pieces of 64 scales");
  static constexpr int kOut = TN * TM * (int)sizeof(T);                // the tile's scores, at the end
  static constexpr int kJoin = (KG - 1) * TN * TM * 4;                 // the other groups' sums, at the end
  static constexpr int kLds = KG * D * kStage > kOut + kJoin ? KG * D * kStage : kOut + kJoin;
  static_assert(D >= 2 && kLds <= 160 * 1024, "the stages fit the LDS");
  static_assert((D - 2) * kLoads < 64, "the wait counter holds the loads in flight");
  static __device__ __forceinline__ int fx(int n) { return (n & 3) | ((n >> (V == 1 ? 2 : 3)) & 1) << 2; }
};

template <int BYTES>
__device__ __forceinline__ void lds_dma(uint32_t dst, uint32_t off, const void* base) {
  static_assert(BYTES == 4 || BYTES == 16, "dword and four-dword pieces");
  // (inline, so that the compiler's own waits leave these loads in flight)
  if constexpr (BYTES == 16)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(__builtin_amdgcn_readfirstlane(dst)), "v"(off), "s"(base) : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(__builtin_amdgcn_readfirstlane(dst)), "v"(off), "s"(base) : "memory");
}
template <typename P>
__device__ __forceinline__ P* uniform(P* p) {
  const uint64_t v = (uint64_t)(uintptr_t)p;
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32));
  return (P*)(uintptr_t)(((uint64_t)hi << 32) | lo);
}

// value K of a row of 16 lanes, in all of them
template <int K>
__device__ __forceinline__ float row_bcast(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x150 + K, 0xf, 0xf, true));
}

// Workgroup -> tile: each XCD takes one contiguous run of tiles (its L2 then holds their rows), in
// which up to 8 query tiles pass over the item tiles together.
__device__ __forceinline__ void tile_of(int L, int total, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int xcd = L & 7, q8 = total >> 3, r8 = total & 7;
  const int i = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + (L >> 3);
  const int band = i / (8 * tiles_n), m0 = band * 8, rows = tiles_m - m0 < 8 ? tiles_m - m0 : 8;
  const int j = i - band * 8 * tiles_n;
  tm = m0 + j % rows;
  tn = j / rows;
}

template <typename T, bool TILE, int WN, int WM, int MT, int D, int KG>
__global__ __launch_bounds__(KG* WN* WM * 64, KG* WN* WM > 8 ? KG * WN * WM / 4 : 2) void product_tile_kernel(ProductArgs a, int tiles_m, int tiles_n) {
  using S = TileShape<T, WN, WM, MT, D, KG>;
  constexpr int V = S::V;
  __shared__ __attribute__((aligned(1024))) char smem[S::kLds];
  int tm, tn;
  tile_of(blockIdx.x, gridDim.x, tiles_m, tiles_n, tm, tn);
  const int64_t n0 = (int64_t)tn * S::TN, m0 = (int64_t)tm * S::TM;
  const int all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = all / S::kWaves, wave = all % S::kWaves;
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wn = wave % WN, wm = wave / WN;
  const int nx = (int)(a.N - n0 < S::TN ? a.N - n0 : S::TN), nq = (int)(a.M - m0 < S::TM ? a.M - m0 : S::TM);

  // this lane's source offsets (rows past the end repeat the last one; the host keeps 256 rows under 2^32 bytes)
  uint32_t xoff[S::kXP], qoff[S::kQP];
#pragma unroll
  for (int p = 0; p < S::kXP; ++p) {
    const int row = (wave * S::kXP + p) * 8 + (lane >> 3);
    xoff[p] = (uint32_t)(row < nx ? row : nx - 1) * (uint32_t)a.ldx + (((lane & 7) ^ S::fx(row)) << 4);
  }
#pragma unroll
  for (int p = 0; p < S::kQP; ++p) {
    const int row = (wave * S::kQP + p) * 8 + (lane >> 3);
    qoff[p] = (uint32_t)(row < nq ? row : nq - 1) * (uint32_t)a.ldq + (((lane & 7) ^ (row & 7)) << 4);
  }
  const uint8_t* xb = uniform(a.x + n0 * a.ldx);
  const uint8_t* qb = uniform(a.q + m0 * a.ldq);
  const float* xsb = uniform(a.xs + (TILE ? n0 / kBlock : n0));
  const float* qsb = uniform(a.qs + m0);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem + group * D * S::kStage;
  auto stage = [&](int b, int buf) __attribute__((always_inline)) {
    const uint32_t at = lds0 + buf * S::kStage;
    const uint8_t* x = xb + (int64_t)b * kBlock;
    const uint8_t* q = qb + (int64_t)b * kBlock;
#pragma unroll
    for (int p = 0; p < S::kXP; ++p) lds_dma<16>(at + (wave * S::kXP + p) * 1024, xoff[p], x);
#pragma unroll
    for (int p = 0; p < S::kQP; ++p) lds_dma<16>(at + S::kX + (wave * S::kQP + p) * 1024, qoff[p], q);
    // (every wave issues the same number, so that one count waits for a stage: the last pieces may repeat)
#pragma unroll
    for (int j = 0; j < S::kSP; ++j) {
      const int i = (j * S::kWaves + wave) % ((S::TN + S::TM) / 64);
      if (i < S::TN / 64) {
        const int row = i * 64 + lane, n = row < nx ? row : nx - 1;
        lds_dma<4>(at + S::kX + S::kQ + i * 256, (uint32_t)(TILE ? n / kBlock : n) * 4, xsb + b * a.ldxs);
      } else {
        const int row = (i - S::TN / 64) * 64 + lane;
        lds_dma<4>(at + S::kX + S::kQ + i * 256, (uint32_t)(row < nq ? row : nq - 1) * 4, qsb + b * a.ldqs);
      }
    }
  };

  // this lane's places in a stage
  uint32_t xat[4], qat;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int row = wn * 64 + (t / V) * 16 * V + (r >> 2) * 4 * V + (t % V) * 4 + (r & 3);
    xat[t] = row * kBlock + ((g ^ S::fx(row)) << 4);
  }
  qat = S::kX + (wm * MT * 16 + r) * kBlock + ((g ^ (r & 7)) << 4);

  f32x4 acc[MT][4] = {};
  // Group `group` of KG takes blocks group, group + KG, ...; its step i is block i KG + group.  D stages a group:
  // while a step is computed, the next D - 1 are in flight.
  auto block = [&](int i) { return i * KG + group; };
#pragma unroll
  for (int i = 0; i < D - 1; ++i)
    if (block(i) < a.kb) stage(block(i), i);
  int cur = 0;
  for (int i0 = 0; i0 * KG < a.kb; ++i0) {
    if (D > 2 && block(i0 + D - 2) < a.kb)
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"((D - 2) * S::kLoads) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();  // this step's block is in for every wave, and the stage of the step before is free
    if (block(i0 + D - 1) < a.kb) stage(block(i0 + D - 1), cur == 0 ? D - 1 : cur - 1);
    if (KG > 1 && block(i0) >= a.kb) break;  // (the last step, for the groups without a block in it)
    const char* at = smem + group * D * S::kStage + cur * S::kStage;
    cur = cur + 1 == D ? 0 : cur + 1;
    const float* sc = (const float*)(at + S::kX + S::kQ);
    typedef typename Mode<T>::Frag Frag;
    Frag x[4], q;
    f32x4 sx[4], p[3];
    float sq[MT];
    auto load_q = [&](int mt) __attribute__((always_inline)) {
      const char* qp = at + mt * 16 * kBlock;
      return Mode<T>::make(*(const u32x4*)(qp + qat), *(const u32x4*)(qp + (qat ^ 64)));
    };
    q = load_q(0);
#pragma unroll
    for (int t = 0; t < 4; ++t) x[t] = Mode<T>::make(*(const u32x4*)(at + xat[t]), *(const u32x4*)(at + (xat[t] ^ 64)));
    float s1 = 0.f;
    if constexpr (TILE) s1 = sc[wn * 64];  // (64 items of one tile)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) sq[mt] = sc[S::TN + wm * MT * 16 + mt * 16 + r];
    if constexpr (!TILE) {
#pragma unroll
      for (int t = 0; t < 4; ++t) sx[t] = *(const f32x4*)(sc + wn * 64 + (t / V) * 16 * V + g * 4 * V + (t % V) * 4);
    }
    // product i is scaled and added two products later, when it is ready
    auto add = [&](int i) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float f = TILE ? sq[i / 4] : sq[i / 4] * sx[i % 4][j];
        acc[i / 4][i % 4][j] = fmaf(f, p[i % 3][j], acc[i / 4][i % 4][j]);
      }
    };
    if constexpr (TILE) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) sq[mt] *= s1;
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      Frag qn = q;
      if (mt + 1 < MT) qn = load_q(mt + 1);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int i = mt * 4 + t;
        p[i % 3] = Mode<T>::dot(x[t], q);
        if (i >= 2) add(i - 2);
      }
      q = qn;
    }
    add(MT * 4 - 2);
    add(MT * 4 - 1);
  }
  __syncthreads();
  if constexpr (KG > 1) {
    // the groups' sums, added in the groups' order
    f32x4* part = (f32x4*)(smem + S::kOut) + wave * 64 + lane;
    constexpr int kStep = S::kWaves * 64;
    if (group > 0) {
#pragma unroll
      for (int i = 0; i < MT * 4; ++i) part[((group - 1) * MT * 4 + i) * kStep] = acc[i / 4][i % 4];
    }
    __syncthreads();
    if (group == 0) {
#pragma unroll
      for (int w = 0; w < KG - 1; ++w)
#pragma unroll
        for (int i = 0; i < MT * 4; ++i) acc[i / 4][i % 4] += part[(w * MT * 4 + i) * kStep];
    }
  }

  // The results are turned around in the LDS (all reads of the stages are done), so that a store covers
  // 1 KiB of the tile's score rows, each row's part whole: full lines but for a row's two ends.
  constexpr int kRow = S::TN * (int)sizeof(T), kChunks = kRow / 16;  // bytes and 16-byte chunks of a row
  constexpr int kSwz = kChunks < 16 ? kChunks - 1 : 15;
  static_assert(kChunks <= 64, "a store covers whole rows");
  typedef T Out __attribute__((ext_vector_type(4 * V)));
  typedef T OutAt __attribute__((ext_vector_type(4 * V), aligned(sizeof(T))));
  if (KG == 1 || group == 0) {
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    char* row = smem + (wm * MT * 16 + mt * 16 + r) * kRow;
#pragma unroll
    for (int u = 0; u < 4 / V; ++u) {
      Out v;
#pragma unroll
      for (int j = 0; j < 4 * V; ++j) v[j] = (T)acc[mt][u * V + (j >> 2)][j & 3];
      *(Out*)(row + (((wn * 16 / V + u * 4 + g) ^ (r & kSwz)) << 4)) = v;
    }
  }
  }
  __syncthreads();
  const int c = threadIdx.x & (kChunks - 1);
  const int64_t n = n0 + c * 4 * V;
  if (n >= a.N) return;
  constexpr int kRows = S::kThreads / kChunks;  // rows of one store by all threads
#pragma unroll
  for (int i = 0; i < (S::TM + kRows - 1) / kRows; ++i) {
    const int row = i * kRows + threadIdx.x / kChunks;
    const int64_t m = m0 + row;
    if (row >= S::TM || m >= a.M) break;
    const Out v = *(const Out*)(smem + row * kRow + ((c ^ (row & kSwz)) << 4));
    T* p = (T*)a.out + m * a.ldo + n;
    if (n + 4 * V <= a.N) {
      __builtin_nontemporal_store(OutAt(v), (OutAt*)p);
    } else {
#pragma unroll
      for (int j = 0; j < 4 * V; ++j)
        if (n + j < a.N) p[j] = v[j];
    }
  }
}

// ---- bf16 scores of many rows: one workgroup a CU, tile after tile --------------------------------
// Tiles of 256 x 256, 8 waves of 64 items x 128 queries, two stages.  What the LDS has to deliver bounds it
// (192 KB a block to the 8 waves, beside 64 KB that come in), then the matrix cores, then the scaling (4 or 8
// FMA slots beside each product of 16 x 16 x 128).  Hence:
//  - a block's last two query tiles are multiplied item tile by item tile, and as soon as an item tile is done
//    its registers take the next block's: the burst of reads that opens a block runs beside products;
//  - one barrier a block, before those last products: all reads of the block are done, the next block is in, and
//    the loads of the one after it go out between them (sent earlier, the items' part after a second barrier,
//    they changed nothing beyond the noise);
//  - the loader runs ahead over the tiles' ends, and a tile's scores go out beside the next tile's blocks;
//  - a product is scaled three products later.  The empty asm keeps the compiler from collecting the sums at the
//    end of the block, which would hold all 32 products in registers.
// 4,096 x 8,192 x 4,096: 118 us, 2.33 PFLOP/s (135 us with a workgroup to a tile; 3.2 PFLOP/s is what a large 8-bit
// product without block scales reaches).  4,096 x 125,000 x 768, whose rows begin anywhere in a line, measured in turn: 625 us
// against 743 with tiles of 128 and 722 with 128 bytes of a row to a store; with 124,992 items, whose rows begin at
// lines, 128 bytes take 545 us and 512 take 615.  (506 us over the same tensors again and again, 655 over inputs that change.)
// The clock falls to 2.0 to 2.1 GHz under this load (2.4 without): the same product of rows that are all alike, whose
// wires hardly switch, is 12 to 16 % faster.
template <typename T>
using RunShape = TileShape<T, 4, 2, 8, 2, 1>;  // 256 x 256
constexpr int kCus = 256;

template <typename T, bool TILE, bool LINES>
__global__ __launch_bounds__(512, 2) void product_run_kernel(ProductArgs a, int tiles_m, int tiles_n) {
  using S = RunShape<T>;
  constexpr int V = S::V, WN = 4, MT = 8;
  static_assert(std::is_same_v<Mode<T>, Narrow> && V == 2 && S::kThreads == 512, "bf16 scores");
  constexpr int kOwn = LINES ? 16 * 64 * 2 : 0;  // a wave's 16 x 64 scores
  static_assert(2 * S::kStage + S::kWaves * kOwn <= 160 * 1024, "the stages and the waves' turning places fit the LDS");
  __shared__ __attribute__((aligned(1024))) char smem[2 * S::kStage + S::kWaves * kOwn];
  const int total = tiles_m * tiles_n;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wn = wave % WN, wm = wave / WN;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem;

  // the loader: the next block of the next tile to go to the LDS
  int d_tile = blockIdx.x, d_b = 0;
  uint32_t xoff[S::kXP], qoff[S::kQP], soff[S::kSP];
  const uint8_t *xb, *qb;
  const float *xsb, *qsb;
  // (where rows do not begin at lines there are no registers left for what a tile's start and end derive from the
  // lane: the empty asm has it worked out there instead of kept, and spilled, over the blocks)
  auto aim = [&]() __attribute__((always_inline)) {
    int tm, tn, ln = lane;
    if constexpr (!LINES) asm volatile("" : "+v"(ln));
    tile_of(d_tile, total, tiles_m, tiles_n, tm, tn);
    const int64_t n0 = (int64_t)tn * S::TN, m0 = (int64_t)tm * S::TM;
    const int nx = (int)(a.N - n0 < S::TN ? a.N - n0 : S::TN), nq = (int)(a.M - m0 < S::TM ? a.M - m0 : S::TM);
#pragma unroll
    for (int p = 0; p < S::kXP; ++p) {
      const int row = (wave * S::kXP + p) * 8 + (ln >> 3);
      xoff[p] = (uint32_t)(row < nx ? row : nx - 1) * (uint32_t)a.ldx + (((ln & 7) ^ S::fx(row)) << 4);
    }
#pragma unroll
    for (int p = 0; p < S::kQP; ++p) {
      const int row = (wave * S::kQP + p) * 8 + (ln >> 3);
      qoff[p] = (uint32_t)(row < nq ? row : nq - 1) * (uint32_t)a.ldq + (((ln & 7) ^ (row & 7)) << 4);
    }
#pragma unroll
    for (int j = 0; j < S::kSP; ++j) {
      const int i = (j * S::kWaves + wave) % ((S::TN + S::TM) / 64);
      const int row = (i < S::TN / 64 ? i : i - S::TN / 64) * 64 + ln, n = i < S::TN / 64 ? nx : nq;
      const int c = row < n ? row : n - 1;
      soff[j] = (uint32_t)(TILE && i < S::TN / 64 ? c / kBlock : c) * 4;
    }
    xb = a.x + n0 * a.ldx;
    qb = a.q + m0 * a.ldq;
    xsb = a.xs + (TILE ? n0 / kBlock : n0);
    qsb = a.qs + m0;
  };
  // load i of the S::kLoads that bring the loader's block into stage `buf`
  auto load = [&](int i, int buf) __attribute__((always_inline)) {
    const uint32_t at = lds0 + buf * S::kStage;
    if (i < S::kXP) {
      lds_dma<16>(at + (wave * S::kXP + i) * 1024, xoff[i], uniform(xb + (int64_t)d_b * kBlock));
    } else if (i < S::kXP + S::kQP) {
      i -= S::kXP;
      lds_dma<16>(at + S::kX + (wave * S::kQP + i) * 1024, qoff[i], uniform(qb + (int64_t)d_b * kBlock));
    } else {
      const int j = i - S::kXP - S::kQP, piece = (j * S::kWaves + wave) % ((S::TN + S::TM) / 64);
      const float* base = piece < S::TN / 64 ? xsb + d_b * a.ldxs : qsb + d_b * a.ldqs;
      lds_dma<4>(at + S::kX + S::kQ + piece * 256, soff[j], uniform(base));
    }
  };
  auto loaded = [&]() __attribute__((always_inline)) {
    if (++d_b == a.kb) {
      d_b = 0;
      d_tile += gridDim.x;
      if (d_tile < total) aim();
    }
  };
  auto load_next = [&](int buf) __attribute__((always_inline)) {
    if (d_tile >= total) return;
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) load(i, buf);
    loaded();
  };

  auto x_tile = [](int t) { return ((t / V) * 16 * V + (t % V) * 4) * kBlock; };
  const int xrow = wn * 64 + (r >> 2) * 4 * V + (r & 3);
  const uint32_t xat = xrow * kBlock + ((g ^ S::fx(xrow)) << 4);
  const uint32_t qat = S::kX + (wm * MT * 16 + r) * kBlock + ((g ^ (r & 7)) << 4);
  auto load_x = [&](const char* at, int t) __attribute__((always_inline)) {
    return Narrow::make(*(const u32x4*)(at + xat + x_tile(t)), *(const u32x4*)(at + (xat ^ 64) + x_tile(t)));
  };
  auto load_q = [&](const char* at, int mt) __attribute__((always_inline)) {
    return Narrow::make(*(const u32x4*)(at + qat + mt * 16 * kBlock), *(const u32x4*)(at + (qat ^ 64) + mt * 16 * kBlock));
  };
  constexpr int kTail = 2, LAG = 3;

  aim();
  load_next(0);
  load_next(1);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  i32x8 x[4], qr[2];
  qr[0] = load_q(smem, 0);
#pragma unroll
  for (int t = 0; t < 4; ++t) x[t] = load_x(smem, t);
  int cur = 0;
  for (int tile = blockIdx.x; tile < total; tile += gridDim.x) {
    f32x4 acc[MT][4] = {};
    for (int b = 0; b < a.kb; ++b) {
      const char* at = smem + cur * S::kStage;
      const char* nat = smem + (cur ^ 1) * S::kStage;
      const float* sc = (const float*)(at + S::kX + S::kQ);
      i32x8 q[MT];
      float sq[MT], sxv;
      f32x4 p[LAG + 1];
      sxv = TILE ? sc[wn * 64] : sc[wn * 64 + (r / (4 * V)) * 16 * V + g * 4 * V + ((r >> 2) % V) * 4 + (r & 3)];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) sq[mt] = sc[S::TN + wm * MT * 16 + mt * 16 + r];
      qr[1] = load_q(at, 1);
      q[0] = qr[0];
      if constexpr (TILE) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) sq[mt] *= sxv;
      }
      auto qi = [](int i) { return i < (MT - kTail) * 4 ? i / 4 : MT - kTail + (i - (MT - kTail) * 4) % kTail; };
      auto xi = [](int i) { return i < (MT - kTail) * 4 ? i % 4 : (i - (MT - kTail) * 4) / kTail; };
      auto add = [&](int i) __attribute__((always_inline)) {
        const int mt = qi(i), t = xi(i);
        const float s = sq[mt];
        f32x4 f = {s, s, s, s};
        if constexpr (!TILE) {
          if (t == 0) f = f32x4{row_bcast<0>(sxv) * s, row_bcast<1>(sxv) * s, row_bcast<2>(sxv) * s, row_bcast<3>(sxv) * s};
          if (t == 1) f = f32x4{row_bcast<4>(sxv) * s, row_bcast<5>(sxv) * s, row_bcast<6>(sxv) * s, row_bcast<7>(sxv) * s};
          if (t == 2) f = f32x4{row_bcast<8>(sxv) * s, row_bcast<9>(sxv) * s, row_bcast<10>(sxv) * s, row_bcast<11>(sxv) * s};
          if (t == 3) f = f32x4{row_bcast<12>(sxv) * s, row_bcast<13>(sxv) * s, row_bcast<14>(sxv) * s, row_bcast<15>(sxv) * s};
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[mt][t][j] = fmaf(f[j], p[i % (LAG + 1)][j], acc[mt][t][j]);
        asm volatile("" : "+v"(acc[mt][t]));
      };
#pragma unroll
      for (int i = 0; i < MT * 4; ++i) {
        const int mt = qi(i), t = xi(i);
        if (i == (MT - kTail) * 4) {
          q[MT - 1] = qr[(MT - 1) & 1];
          asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
        }
        p[i % (LAG + 1)] = Narrow::dot(x[t], q[mt]);
        // the loads of the block after the next go out between these last products
        if (i >= (MT - kTail) * 4 && (LINES || b + 1 < a.kb) && d_tile < total) {
          constexpr int n = kTail * 4;
          const int k = i - (MT - kTail) * 4;
#pragma unroll
          for (int l = k * S::kLoads / n; l < (k + 1) * S::kLoads / n; ++l) load(l, cur);
        }
        if (i < (MT - kTail) * 4) {
          if (t == 0 && mt + 1 < MT) q[mt + 1] = qr[(mt + 1) & 1];
          if (t == 1 && mt + 2 < MT) qr[mt & 1] = load_q(at, mt + 2);
        } else if ((i - (MT - kTail) * 4) % kTail == kTail - 1) {
          x[t] = load_x(nat, t);  // (after the last block of all: an old stage's, unused)
          if (t == 0) qr[0] = load_q(nat, 0);
        }
        if (i >= LAG) add(i - LAG);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int i = MT * 4 - LAG; i < MT * 4; ++i) add(i);
      if ((LINES || b + 1 < a.kb) && d_tile < total) loaded();
      cur ^= 1;
    }

    int tm, tn;
    tile_of(tile, total, tiles_m, tiles_n, tm, tn);
    typedef T Out __attribute__((ext_vector_type(8)));
    typedef T OutAt __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    if constexpr (LINES) {
      // A wave turns 16 of its rows at a time around in a place of its own: a store covers 128 bytes of 8 rows, a
      // whole line of each, while the next tile's two first blocks come in.
      const int64_t n0 = (int64_t)tn * S::TN + wn * 64, m0 = (int64_t)tm * S::TM + wm * MT * 16;
      char* own = smem + 2 * S::kStage + wave * kOwn;
      const int64_t n = n0 + (lane & 7) * 8;
      T* out = (T*)a.out + (m0 + (lane >> 3)) * a.ldo + n;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          Out v;
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = (T)acc[mt][u * 2 + (j >> 2)][j & 3];
          *(Out*)(own + r * 128 + (((u * 4 + g) ^ (r & 7)) << 4)) = v;
        }
        __builtin_amdgcn_wave_barrier();  // (a wave's LDS accesses are in order; this keeps the compiler's so)
        asm volatile("" ::: "memory");
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = h * 8 + (lane >> 3);
          const Out v = *(const Out*)(own + row * 128 + (((lane & 7) ^ (row & 7)) << 4));
          if (m0 + mt * 16 + row < a.M) {
            T* p = out + (int64_t)(mt * 16 + h * 8) * a.ldo;
            if (n + 8 <= a.N) {
              __builtin_nontemporal_store(OutAt(v), (OutAt*)p);
            } else {
#pragma unroll
              for (int j = 0; j < 8; ++j)
                if (n + j < a.N) p[j] = v[j];
            }
          }
        }
        __builtin_amdgcn_wave_barrier();
        asm volatile("" ::: "memory");
      }
    } else {
      // Rows that do not begin at a line: 128 bytes of a row are parts of two lines, and parts of lines written past
      // the L2 cost twice.  The scores are turned around in the last block's stage, half the tile's queries at a
      // time, so that a store covers 512 bytes of a row; the stage is loaded again after that.
      constexpr int kRow = S::TN * 2, kHalf = S::TM / 2;
      static_assert(kHalf * kRow <= S::kStage && kRow == 512, "half a tile's scores fit a stage");
      char* turn = smem + (cur ^ 1) * S::kStage;
      int tid = threadIdx.x;
      asm volatile("" : "+v"(tid));
      const int c = tid & 31;
      const int64_t n = (int64_t)tn * S::TN + c * 8;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < MT / 2; ++i) {
          char* row = turn + (wm * (kHalf / 2) + i * 16 + (tid & 15)) * kRow;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            Out v;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = (T)acc[h * (MT / 2) + i][u * 2 + (j >> 2)][j & 3];
            *(Out*)(row + (((wn * 8 + u * 4 + (tid >> 4 & 3)) ^ (tid & 15)) << 4)) = v;
          }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kHalf / 16; ++i) {
          const int row = i * 16 + (tid >> 5);
          const int64_t m = (int64_t)tm * S::TM + (row / (kHalf / 2)) * (S::TM / 2) + h * (kHalf / 2) + row % (kHalf / 2);
          const Out v = *(const Out*)(turn + row * kRow + ((c ^ (row & 15)) << 4));
          if (m < a.M) {
            T* p = (T*)a.out + m * a.ldo + n;
            if (n + 8 <= a.N) {
              __builtin_nontemporal_store(OutAt(v), (OutAt*)p);
            } else {
#pragma unroll
              for (int j = 0; j < 8; ++j)
                if (n + j < a.N) p[j] = v[j];
            }
          }
        }
        __syncthreads();
      }
      load_next(cur ^ 1);
    }
  }
}

// ---- which kernel ---------------------------------------------------------------------------
int too_many() { return abi_fail(BB_E_ARG, "bb_scores_fp8: too many scores for one call"); }

template <typename T, int KS, int PF>
int launch_few(const ProductArgs& a, void* stream) {
  const int64_t n_groups = (a.N + 15) / 16, total = n_groups * ((a.M + 15) / 16);
  if (total > (int64_t)(0xFFFFFFFFu / (KS * 64))) return too_many();
  return abi_launch("bb_scores_fp8", product_few_kernel<T, KS, PF>, dim3((uint32_t)total), dim3(KS * 64), 0,
                    (hipStream_t)stream, a, (int)n_groups);
}

template <typename T, int WN, int WM, int MT, int D, int KG>
int launch_tile(const ProductArgs& a, void* stream) {
  using S = TileShape<T, WN, WM, MT, D, KG>;
  const int64_t tiles_m = (a.M + S::TM - 1) / S::TM, tiles_n = (a.N + S::TN - 1) / S::TN;
  if (tiles_m * tiles_n > (int64_t)(0xFFFFFFFFu / S::kThreads)) return too_many();
  return abi_launch("bb_scores_fp8",
                    a.tile ? product_tile_kernel<T, true, WN, WM, MT, D, KG> : product_tile_kernel<T, false, WN, WM, MT, D, KG>,
                    dim3((uint32_t)(tiles_m * tiles_n)), dim3(S::kThreads), 0, (hipStream_t)stream, a, (int)tiles_m,
                    (int)tiles_n);
}

template <typename T>
int launch_run(const ProductArgs& a, void* stream) {
  using S = RunShape<T>;
  const int64_t tiles_m = (a.M + S::TM - 1) / S::TM, tiles_n = (a.N + S::TN - 1) / S::TN, total = tiles_m * tiles_n;
  if (total > 0x7FFFFFFF / 2) return too_many();
  const bool lines = (uintptr_t)a.out % 128 == 0 && a.ldo % 64 == 0;
  return abi_launch("bb_scores_fp8", lines ? (a.tile ? product_run_kernel<T, true, true> : product_run_kernel<T, false, true>)
                                           : (a.tile ? product_run_kernel<T, true, false> : product_run_kernel<T, false, false>),
                    dim3((uint32_t)(total < kCus ? total : kCus)), dim3(S::kThreads), 0, (hipStream_t)stream, a, (int)tiles_m,
                    (int)tiles_n);
}

inline int64_t tiles(const ProductArgs& a, int t) { return ((a.M + t - 1) / t) * ((a.N + t - 1) / t); }
inline int64_t up(int64_t x, int64_t by) { return (x + by - 1) / by; }

// Times below: M x N x K on one MI355X, kernel alone, "against" = the other choice.
template <typename T>
int launch_product(const ProductArgs& a, void* stream) {
  // The tiles' source offsets are 32-bit within 256 rows; rows further apart are read by their 64-bit addresses.
  const bool far = a.ldx >= (1 << 24) || a.ldq >= (1 << 24);
  const bool split = tiles(a, 64) <= kCus && a.kb >= 8;  // fewer 64 x 64 tiles than CUs, and long rows: split the rows
  bool few = a.M <= 16;
  // 9 to 16 rows waste less of a tile: against a long list of items it reads them in larger pieces (16 x 50,000 x 1,024
  // 10.9 us against 15.2; 1 x 100,000 x 768 19.1 against 15.5), and against 6,144 to 16,384 items long rows are
  // better split in it (16 x 8,192 x 4,096 10.1 us against 12.0; 16 x 4,096 x 4,096 9.7 against 7.1)
  if (a.M > 8 && a.M <= 16) few = !(a.N >= 32768 || (split && tiles(a, 64) >= 96));
  // few scores and long rows: 20 x 300 x 8,192 9.8 us against 24.9; 64 x 2,048 x 4,096 (512) 10.4 against 8.8
  if (a.M > 16 && split && tiles(a, 16) <= 256) few = true;
  if (few || far) {
    if (a.kb == 1) return launch_few<T, 1, 1>(a, stream);
    // one block a wave: 1 x 25,216 x 384 4.1 us against 8.3 with 8 waves of two
    if (a.kb <= 8) return launch_few<T, 4, 1>(a, stream);
    // two blocks of a wave in flight need the registers of other workgroups: 4 x 20,000 x 2,048 10.1 us with one
    // against 13.7, 16 x 4,096 x 4,096 8.3 against 7.1
    return a.N > 16384 ? launch_few<T, 8, 1>(a, stream) : launch_few<T, 8, 2>(a, stream);
  }
  // 64 x 8,192 x 4,096 10.9 us against 13.0 unsplit, 128 x 2,048 x 8,192 17.4 against 23.2
  if (split) return launch_tile<T, 1, 4, 1, 2, 4>(a, stream);
  if (a.M <= 64 || tiles(a, 128) < 192) {
    // three stages where no CU has more than two workgroups, so that there is LDS for them, and rows are long:
    // 128 x 16,384 x 4,096 16.8 us against 19.7, 64 x 32,768 x 8,192 57.5 against 64.7; 64 x 65,536 x 2,048 (four
    // a CU) 31.7 against 30.0, 64 x 30,000 x 1,536 10.7 against 10.2; f32 and f16 scores are bound by the matrix cores (12.9
    // against 13.6)
    if constexpr (std::is_same_v<T, __bf16>) {
      if (a.kb >= 16 && tiles(a, 64) <= 2 * kCus) return launch_tile<T, 1, 4, 1, 3, 1>(a, stream);
    }
    // 40 x 100,000 x 384 f32 14.6 us against 18.6 with tiles of 128; 256 x 8,192 x 512 (128 tiles) 4.9 against 6.4
    return launch_tile<T, 1, 4, 1, 2, 1>(a, stream);
  }
  // About one tile of 128 a CU: halves of them, two workgroups to a CU, overlap.  333 x 10,007 x 1,000 (237 tiles) bf16 9.7 us
  // against 11.2, f16 13.2 against 14.0, 512 x 8,192 x 4,096 (256) bf16 24.2 against 28.0, f16 41.1 against 39.8,
  // 300 x 12,000 x 384 (282) 6.5 against 7.4, 128 x 25,216 x 384 f32 (197) 7.8 against 8.0; 768 x 8,192 x 4,096 (384) bf16
  // 36.0 against 35.0, f16 61.4 against 58.9, 512 x 16,384 x 768 (512) bf16 13.7 against 12.2, f16 18.2 against 14.9
  if (4 * tiles(a, 128) <= 5 * kCus) return launch_tile<T, 1, 4, 2, 2, 1>(a, stream);
  if constexpr (std::is_same_v<T, __bf16>) {
    // rounds over the chip: one 256 x 256 tile a CU takes 1.8 times what two 128 x 128 tiles a CU do (4,096 x 8,192 x 4,096:
    // 2 rounds 118 us against 4 rounds 135; 1,024 x 8,192 x 8,192: half a round 98 us against one 74).  A single
    // round has no tile after it to overlap with, and pays for long rows alone (2,048 x 8,192 x 4,096 63.5 us against
    // 76.0, x 512 18.2 against 16.7; 333 x 25,216 x 384 14.9 against 10.8)
    const int64_t rounds = up(tiles(a, 256), kCus);
    if (9 * rounds <= 5 * up(tiles(a, 128), 2 * kCus) && (rounds > 1 || a.kb >= 12)) return launch_run<T>(a, stream);
  }
  return launch_tile<T, 2, 2, 4, 2, 1>(a, stream);
}

int check_rows(const bb_fp8_rows* r, const std::string& what) {
  auto bad = [&](const char* why) { return abi_fail(BB_E_ARG, what + why); };
  if (!r) return bad(" is null");
  if (r->rows < 0 || r->d < 0) return bad(" has a negative size");
  if (r->rows > 0x7FFFFFFF || r->d > (1 << 24)) return bad(" has 2^31 rows or more, or rows over 2^24 wide");
  if (r->rows == 0 || r->d == 0) return BB_OK;
  if (!r->codes || !r->scales) return bad(" has null codes or scales");
  if ((uintptr_t)r->codes % 16 || r->ld % 16) return bad("' codes or their ld are not 16-byte aligned");
  if ((uintptr_t)r->scales % 4) return bad("' scales are not aligned");
  if (r->ld < blocks_of(r->d) * kBlock) return bad("' ld is below d rounded up to 128");
  if (r->scales_ld < (r->tile ? blocks_of(r->rows) : r->rows)) return bad("' scales_ld is below the scales of a block column");
  return BB_OK;
}

// bytes from the first to the last of n rows
inline uint64_t span(int64_t n, int64_t ld, int64_t width, int es) { return ((uint64_t)(n - 1) * ld + width) * es; }
// whether [p, p + bytes) meets the rows' codes or scales
inline bool meets(const bb_fp8_rows* r, const void* p, uint64_t bytes) {
  const int64_t kb = blocks_of(r->d);
  return overlap(r->codes, span(r->rows, r->ld, kb * kBlock, 1), p, bytes) ||
         overlap(r->scales, span(kb, r->scales_ld, r->tile ? blocks_of(r->rows) : r->rows, 4), p, bytes);
}

inline int elem(int dtype) { return dtype == BB_F32 ? 4 : dtype == BB_BF16 || dtype == BB_F16 ? 2 : 0; }

}  // namespace
}  // namespace bb

extern "C" int bb_quantize_fp8(int32_t device, const void* x, int32_t dtype, int64_t ldx, const bb_fp8_rows* out,
                               void* stream) {
  using namespace bb;
  return abi_call("bb_quantize_fp8", [&]() -> int {
    int rc = check_rows(out, "bb_quantize_fp8: out");
    if (rc) return rc;
    const int es = elem(dtype);
    if (!es) return abi_fail(BB_E_ARG, "bb_quantize_fp8: dtype must be BB_F32, BB_BF16 or BB_F16");
    if (out->rows == 0 || out->d == 0) return BB_OK;
    if (!x) return abi_fail(BB_E_ARG, "bb_quantize_fp8: null rows");
    if ((uintptr_t)x % es) return abi_fail(BB_E_ARG, "bb_quantize_fp8: rows are not aligned to their type");
    if (ldx < out->d && out->rows > 1) return abi_fail(BB_E_ARG, "bb_quantize_fp8: ldx < d");
    if (meets(out, x, span(out->rows, out->rows > 1 ? ldx : 0, out->d, es)))
      return abi_fail(BB_E_ARG, "bb_quantize_fp8: out overlaps the rows");
    if (overlap(out->codes, span(out->rows, out->ld, blocks_of(out->d) * kBlock, 1), out->scales,
                span(blocks_of(out->d), out->scales_ld, out->tile ? blocks_of(out->rows) : out->rows, 4)))
      return abi_fail(BB_E_ARG, "bb_quantize_fp8: codes and scales overlap");
    CallDevice dev;
    if ((rc = dev.enter(device, "bb_quantize_fp8"))) return rc;
    QuantArgs a{x, ldx, out->rows, out->d, out->codes, out->ld, out->scales, out->scales_ld, (int32_t)blocks_of(out->d)};
    const int64_t groups = out->tile ? blocks_of(a.n) : (a.n + kQRows - 1) / kQRows;
    if (groups * a.kb > 0xFFFFFFFFll / 512) return abi_fail(BB_E_ARG, "bb_quantize_fp8: too many rows for one call");
    auto go = [&](auto rows_kernel, auto tiles_kernel) {
      return abi_launch("bb_quantize_fp8", out->tile ? tiles_kernel : rows_kernel, dim3((uint32_t)(groups * a.kb)),
                        dim3(512), 0, (hipStream_t)stream, a);
    };
    static_assert(kQRows * 16 == 512, "both kernels run 512 threads");
    if (dtype == BB_F32) return go(quantize_rows_kernel<float>, quantize_tiles_kernel<float>);
    if (dtype == BB_BF16) return go(quantize_rows_kernel<__bf16>, quantize_tiles_kernel<__bf16>);
    return go(quantize_rows_kernel<_Float16>, quantize_tiles_kernel<_Float16>);
  });
}

extern "C" int bb_scores_fp8(int32_t device, const bb_fp8_rows* q, const bb_fp8_rows* items, void* out, int32_t dtype,
                             int64_t ldo, void* stream) {
  using namespace bb;
  return abi_call("bb_scores_fp8", [&]() -> int {
    int rc;
    if ((rc = check_rows(q, "bb_scores_fp8: queries")) || (rc = check_rows(items, "bb_scores_fp8: items"))) return rc;
    auto bad = [&](const char* why) { return abi_fail(BB_E_ARG, std::string("bb_scores_fp8: ") + why); };
    const int es = elem(dtype);
    if (!es) return bad("dtype must be BB_F32, BB_BF16 or BB_F16");
    if (q->d != items->d) return bad("queries and items differ in width");
    if (q->d == 0) return bad("rows of width 0");
    if (q->tile) return bad("queries have a scale for each row and block");
    if (q->rows == 0 || items->rows == 0) return BB_OK;
    if (!out) return bad("null out");
    if ((uintptr_t)out % es) return bad("out is not aligned to its type");
    if (ldo < items->rows && q->rows > 1) return bad("ldo is below the number of items");
    const uint64_t bytes = span(q->rows, q->rows > 1 ? ldo : 0, items->rows, es);
    if (meets(q, out, bytes) || meets(items, out, bytes)) return bad("out overlaps the queries or the items");
    CallDevice dev;
    if ((rc = dev.enter(device, "bb_scores_fp8"))) return rc;
    ProductArgs a{q->codes, items->codes, q->scales, items->scales, q->ld, items->ld, q->scales_ld, items->scales_ld,
                  out, ldo, q->rows, items->rows, (int32_t)blocks_of(q->d), items->tile != 0};
    return dtype == BB_F32 ? launch_product<float>(a, stream) : dtype == BB_BF16 ? launch_product<__bf16>(a, stream)
                                                                         : launch_product<_Float16>(a, stream);
  });
}
