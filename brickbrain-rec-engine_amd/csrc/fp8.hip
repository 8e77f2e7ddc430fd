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
// their scales (consecutive in memory) go out as one 128-byte line.
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

// One scale for each 128 x 128 tile: a workgroup holds the tile in registers.
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
//  - 16-bit scores: v_mfma_f32_16x16x128_f8f6f4 on the codes as they are.  It cuts each product of a
//    group of 8 (8 consecutive bytes of a lane) at 2^-13 of the group's largest before it sums
//    them in f32 (measured: the instruction's rounding is not documented; every 8-bit form does the
//    same), an error of 1.4e-5 of the result on normal inputs and at most 2^-10 of the sum of magnitudes.  bf16
//    rounds the result by 2^-8, f16 by 2^-11.
//  - f32 scores: the codes widened to f16, which holds every e4m3 value, and v_mfma_f32_16x16x32_f16,
//    which keeps 24 bits under the largest product (2.9e-9 on the same inputs), at half the rate.
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
using Mode = std::conditional_t<std::is_same_v<T, float>, Wide, Narrow>;

template <typename M>
__device__ __forceinline__ typename M::Frag load32(const uint8_t* p) {
  return M::make(*(const u32x4*)p, *(const u32x4*)(p + 16));
}

// ---- the product of few rows -----------------------------------------------------------------
// Bound by reading the items once: operands go straight from memory to registers, up to PF blocks
// of a wave in flight.  A wave holds 16 NT items x 16 MT queries; the KS waves of a workgroup take every
// KS-th block of the same rows and are summed through LDS, in order of the wave.
template <typename T, int NT, int MT, int KS, int PF>
__global__ __launch_bounds__(KS * 64) void product_few_kernel(ProductArgs a, int n_groups) {
  typedef typename Mode<T>::Frag Frag;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int64_t n0 = (int64_t)(blockIdx.x % n_groups) * 16 * NT, m0 = (int64_t)(blockIdx.x / n_groups) * 16 * MT;
  const uint8_t *xp[NT], *qp[MT];
  const float *xs[NT], *qs[MT];
  const bool whole = n0 + 16 * NT <= a.N;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int64_t n = n0 + t * 16 + r;
    xp[t] = a.x + (n < a.N ? n : a.N - 1) * a.ldx + g * 32;
    const int64_t s = n0 + t * 16 + g * 4;
    xs[t] = a.xs + (a.tile ? n0 / kBlock : s < a.N ? s : a.N - 1);
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int64_t m = m0 + t * 16 + r < a.M ? m0 + t * 16 + r : a.M - 1;
    qp[t] = a.q + m * a.ldq + g * 32;
    qs[t] = a.qs + m;
  }
  f32x4 acc[MT][NT] = {};
  for (int b0 = wave; b0 < a.kb; b0 += KS * PF) {
    u32x4 x[PF][NT][2], q[PF][MT][2];
    f32x4 sx[PF][NT];
    float sq[PF][MT];
#pragma unroll
    for (int f = 0; f < PF; ++f) {
      const int b = b0 + f * KS < a.kb ? b0 + f * KS : b0;  // (a block past the end counts 0 below)
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const u32x4* p = (const u32x4*)(xp[t] + (int64_t)b * kBlock);
        x[f][t][0] = p[0];
        x[f][t][1] = p[1];
      }
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const u32x4* p = (const u32x4*)(qp[t] + (int64_t)b * kBlock);
        q[f][t][0] = p[0];
        q[f][t][1] = p[1];
        sq[f][t] = qs[t][b * a.ldqs];
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float* p = xs[t] + b * a.ldxs;
        if (a.tile) {
          sx[f][t] = f32x4{*p, *p, *p, *p};
        } else if (whole) {
          typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
          sx[f][t] = *(const f32x4u*)p;
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) sx[f][t][j] = n0 + t * 16 + g * 4 + j < a.N ? p[j] : 0.f;
        }
      }
    }
#pragma unroll
    for (int f = 0; f < PF; ++f) {
      if (b0 + f * KS >= a.kb) break;
      Frag xf[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) xf[t] = Mode<T>::make(x[f][t][0], x[f][t][1]);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const Frag qf = Mode<T>::make(q[f][mt][0], q[f][mt][1]);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const f32x4 p = Mode<T>::dot(xf[t], qf);
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[mt][t][j] = fmaf(sq[f][mt] * sx[f][t][j], p[j], acc[mt][t][j]);
        }
      }
    }
  }
  if constexpr (KS > 1) {
    __shared__ f32x4 part[KS - 1][MT * NT][64];
    if (wave > 0) {
#pragma unroll
      for (int i = 0; i < MT * NT; ++i) part[wave - 1][i][lane] = acc[i / NT][i % NT];
    }
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 0; w < KS - 1; ++w)
#pragma unroll
      for (int i = 0; i < MT * NT; ++i) acc[i / NT][i % NT] += part[w][i][lane];
  }
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int64_t m = m0 + mt * 16 + r;
    if (m >= a.M) continue;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      typedef T Out __attribute__((ext_vector_type(4), aligned(sizeof(T))));
      const int64_t n = n0 + t * 16 + g * 4;
      T* p = (T*)a.out + m * a.ldo + n;
      if (n + 4 <= a.N) {
        *(Out*)p = Out{(T)acc[mt][t][0], (T)acc[mt][t][1], (T)acc[mt][t][2], (T)acc[mt][t][3]};
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < a.N) p[j] = (T)acc[mt][t][j];
      }
    }
  }
}

// ---- the product of many rows: tiles staged through LDS ----------------------------------------
// A workgroup of WN x WM waves computes 64 WN items x 16 MT WM queries; a wave 64 items x 16 MT
// queries.  Both operands' blocks of 128 codes go to LDS by LDS-DMA, double buffered: the next
// block's loads are in flight while this one's products run, one barrier to a block.  The block's
// scales go along (4 bytes a row).
//
// LDS rows are 128 bytes of 8 chunks; chunk c of row r sits at position c ^ f(r), with f such that the 8
// rows that 8 neighbouring lanes read together have 8 different f: their 16-byte reads then fall
// on all banks once.  A lane takes chunks g and g + 4 of its row (g = lane >> 4).
//
// Item rows are dealt to MFMA tiles so that a lane's results of V neighbouring tiles are 4 V
// consecutive items: 16-byte stores, 64 bytes of a score row to each 4 lanes.
template <typename T, int WN, int WM, int MT, int D>
struct TileShape {
  static constexpr int kWaves = WN * WM, kThreads = kWaves * 64;
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
  static constexpr int kLds = D * kStage > kOut ? D * kStage : kOut;
  static_assert(D >= 2 && kLds <= 160 * 1024, "the stages fit the LDS");
  static_assert((D - 2) * kLoads < 64, "the wait counter holds the loads in flight");
  static __device__ __forceinline__ int fx(int n) { return (n & 3) | ((n >> (V == 1 ? 2 : 3)) & 1) << 2; }
};

template <int BYTES>
__device__ __forceinline__ void lds_dma(uint32_t dst, uint32_t off, const void* base) {
  static_assert(BYTES == 4 || BYTES == 16, "dword and four-dword pieces");
  // (inline, so that the compiler's own waits leave these loads in flight)
  if constexpr (BYTES == 16)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(dst), "v"(off), "s"(base) : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(dst), "v"(off), "s"(base) : "memory");
}
template <typename P>
__device__ __forceinline__ P* uniform(P* p) {
  const uint64_t v = (uint64_t)(uintptr_t)p;
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32));
  return (P*)(uintptr_t)(((uint64_t)hi << 32) | lo);
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

template <typename T, bool TILE, int WN, int WM, int MT, int D>
__global__ __launch_bounds__(WN* WM * 64, 2) void product_tile_kernel(ProductArgs a, int tiles_m, int tiles_n) {
  using S = TileShape<T, WN, WM, MT, D>;
  constexpr int V = S::V;
  __shared__ __attribute__((aligned(1024))) char smem[S::kLds];
  int tm, tn;
  tile_of(blockIdx.x, gridDim.x, tiles_m, tiles_n, tm, tn);
  const int64_t n0 = (int64_t)tn * S::TN, m0 = (int64_t)tm * S::TM;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
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
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
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
  // D stages: while block b is computed, blocks b + 1 .. b + D - 1 are in flight.  (Past the last block
  // the last one is loaded again, into a stage that nobody reads, so that the count stays the same.)
  auto at_most = [&](int b) { return b < a.kb ? b : a.kb - 1; };
#pragma unroll
  for (int i = 0; i < D - 1; ++i) stage(at_most(i), i);
  int cur = 0;
  for (int b = 0; b < a.kb; ++b) {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((D - 2) * S::kLoads) : "memory");
    __syncthreads();  // block b is in for every wave, and the stage of block b - 1 is free
    stage(at_most(b + D - 1), cur == 0 ? D - 1 : cur - 1);
    const char* at = smem + cur * S::kStage;
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
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();

  // The results are turned around in the LDS (all reads of the stages are done), so that a store covers
  // 1 KiB of the tile's score rows, each row's part whole: full lines but for a row's two ends.
  constexpr int kRow = S::TN * (int)sizeof(T), kChunks = kRow / 16;  // bytes and 16-byte chunks of a row
  constexpr int kSwz = kChunks < 16 ? kChunks - 1 : 15;
  static_assert(kChunks <= 64, "a store covers whole rows");
  typedef T Out __attribute__((ext_vector_type(4 * V)));
  typedef T OutAt __attribute__((ext_vector_type(4 * V), aligned(sizeof(T))));
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
  __syncthreads();
  const int c = threadIdx.x & (kChunks - 1);
  const int64_t n = n0 + c * 4 * V;
  if (n >= a.N) return;
#pragma unroll
  for (int i = 0; i < S::TM * kChunks / S::kThreads; ++i) {
    const int row = i * (S::kThreads / kChunks) + threadIdx.x / kChunks;
    const int64_t m = m0 + row;
    if (m >= a.M) break;
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

// ---- which kernel ---------------------------------------------------------------------------
int too_many() { return abi_fail(BB_E_ARG, "bb_scores_fp8: too many scores for one call"); }

template <typename T, int KS, int PF>
int launch_few(const ProductArgs& a, void* stream) {
  const int64_t n_groups = (a.N + 15) / 16, total = n_groups * ((a.M + 15) / 16);
  if (total > (int64_t)(0xFFFFFFFFu / (KS * 64))) return too_many();
  return abi_launch("bb_scores_fp8", product_few_kernel<T, 1, 1, KS, PF>, dim3((uint32_t)total), dim3(KS * 64), 0,
                    (hipStream_t)stream, a, (int)n_groups);
}

template <typename T, int WN, int WM, int MT, int D>
int launch_tile(const ProductArgs& a, void* stream) {
  using S = TileShape<T, WN, WM, MT, D>;
  const int64_t tiles_m = (a.M + S::TM - 1) / S::TM, tiles_n = (a.N + S::TN - 1) / S::TN;
  if (tiles_m * tiles_n > (int64_t)(0xFFFFFFFFu / S::kThreads)) return too_many();
  return abi_launch("bb_scores_fp8", a.tile ? product_tile_kernel<T, true, WN, WM, MT, D> : product_tile_kernel<T, false, WN, WM, MT, D>,
                    dim3((uint32_t)(tiles_m * tiles_n)), dim3(S::kThreads), 0, (hipStream_t)stream, a, (int)tiles_m,
                    (int)tiles_n);
}

inline int64_t tiles(const ProductArgs& a, int t) { return ((a.M + t - 1) / t) * ((a.N + t - 1) / t); }
inline int64_t up(int64_t x, int64_t by) { return (x + by - 1) / by; }

template <typename T>
int launch_product(const ProductArgs& a, void* stream) {
  // The tiles' source offsets are 32-bit within 256 rows.
  const bool far = a.ldx >= (1 << 24) || a.ldq >= (1 << 24);
  if (a.M <= 16 || far) {
    // one block a wave while it is short (3 blocks, 25,216 items, 1 query: 4.1 us against 8.3 with 8 waves and
    // 6.2 with one), longer rows split over more waves (32 blocks, 8,192 items, 16 queries: 12.1 us against 13.3)
    return a.kb == 1 ? launch_few<T, 1, 1>(a, stream) : a.kb <= 8 ? launch_few<T, 4, 1>(a, stream) : launch_few<T, 8, 2>(a, stream);
  }
  if (tiles(a, 128) < 200) return launch_tile<T, 1, 4, 1, 3>(a, stream);
  if constexpr (sizeof(T) == 2) {
    if (21 * up(tiles(a, 256), 256) <= 11 * up(tiles(a, 128), 512)) return launch_tile<T, 4, 2, 8, 2>(a, stream);
  }
  return launch_tile<T, 2, 2, 4, 2>(a, stream);
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
