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

// 16 consecutive scores of one row from column n, as many as are inside.
template <typename T>
__device__ __forceinline__ void store16(T* row, int64_t n, int64_t N, const f32x4 (&acc)[4]) {
  typedef typename Vec8<T>::type V;
  if (n + 16 <= N) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      V v;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = (T)acc[2 * h + (j >> 2)][j & 3];
      *(V*)(row + n + 8 * h) = v;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (n + j < N) row[n + j] = (T)acc[j >> 2][j & 3];
  }
}

// A wave holds 64 items x 16 queries; operands straight from memory.  Item row p of MFMA tile t
// is item 16 (p >> 2) + 4 t + (p & 3) of the 64, so that a lane's 16 results are 16
// consecutive items of its query.
template <typename T>
__global__ __launch_bounds__(256) void product_kernel(ProductArgs a, int n_groups) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int64_t n0 = ((int64_t)(blockIdx.x % n_groups) * 4 + wave) * 64;
  const int64_t m = (int64_t)(blockIdx.x / n_groups) * 16 + r;
  if (n0 >= a.N) return;
  const int64_t mc = m < a.M ? m : a.M - 1;
  const uint8_t* qp = a.q + mc * a.ldq + g * 32;
  const uint8_t* xp[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int64_t n = n0 + (r >> 2) * 16 + t * 4 + (r & 3);
    xp[t] = a.x + (n < a.N ? n : a.N - 1) * a.ldx + g * 32;
  }
  f32x4 acc[4] = {};
  for (int b = 0; b < a.kb; ++b) {
    const auto q = load32<Mode<T>>(qp + (int64_t)b * kBlock);
    const float sq = a.qs[b * a.ldqs + mc];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const f32x4 p = Mode<T>::dot(load32<Mode<T>>(xp[t] + (int64_t)b * kBlock), q);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t n = n0 + g * 16 + t * 4 + j;
        const float sx = a.xs[b * a.ldxs + (a.tile ? n0 / kBlock : n < a.N ? n : a.N - 1)];
        acc[t][j] = fmaf(sq * sx, p[j], acc[t][j]);
      }
    }
  }
  if (m < a.M) store16((T*)a.out + m * a.ldo, n0 + g * 16, a.N, acc);
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
    const int64_t n_groups = (a.N + 255) / 256, m_groups = (a.M + 15) / 16;
    if (n_groups * m_groups > 0xFFFFFFFFll / 256) return bad("too many scores for one call");
    auto go = [&](auto kernel) {
      return abi_launch("bb_scores_fp8", kernel, dim3((uint32_t)(n_groups * m_groups)), dim3(256), 0,
                        (hipStream_t)stream, a, (int)n_groups);
    };
    if (dtype == BB_F32) return go(product_kernel<float>);
    if (dtype == BB_BF16) return go(product_kernel<__bf16>);
    return go(product_kernel<_Float16>);
  });
}
