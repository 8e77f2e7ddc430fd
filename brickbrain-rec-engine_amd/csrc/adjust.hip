// adjust.hip — penalties for ids seen already, sparse biases and a bit mask on dense scores
// (bb_adjust_scores).
//
// One pass over the scores.  A workgroup takes one chunk of one row: it counts the row's seen
// ids that fall into the chunk in LDS (integer atomics: the order does not matter), keeps the
// position of the last bias entry of each id there (integer max), and then streams the chunk,
// every thread one group of 8 scores at a time.  The row's lists are read again by every chunk of
// the row, from the L2: 4 bytes an entry against 2 x 4096 scores moved.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

#include "abi.h"

namespace bb {
namespace {

constexpr int kThreads = 256;
constexpr int kVec = 8;        // scores per thread and step: 16 bytes of a 16-bit type, a byte of the mask
constexpr int kChunk = 4096;   // scores per workgroup (a multiple of 32: whole mask words)

template <typename T>
struct Vec8 {
  typedef T type __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};

__device__ __forceinline__ int64_t list_id(const void* p, int64_t i, bool wide) {
  return wide ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
}

template <typename T>
__global__ __launch_bounds__(kThreads) void adjust_kernel(bb_adjust a, int n_chunks) {
  extern __shared__ uint32_t lds[];
  const int64_t row = blockIdx.x / n_chunks;
  const int64_t c0 = (int64_t)(blockIdx.x % n_chunks) * kChunk;
  const int len = (int)(a.n - c0 < kChunk ? a.n - c0 : kChunk);
  uint32_t* count = lds;
  uint32_t* slot = lds + (a.seen ? kChunk : 0);
  const int n_words = (a.seen ? kChunk : 0) + (a.bias_ids ? kChunk : 0);
  if (n_words) {
    for (int i = threadIdx.x; i < n_words; i += kThreads) lds[i] = 0;
    __syncthreads();
    if (a.seen) {
      int64_t h = a.n_seen;
      if (a.seen_len) {
        const int64_t l = a.seen_len[row];
        h = l < 0 ? 0 : l < h ? l : h;
      }
      for (int64_t i = threadIdx.x; i < h; i += kThreads) {
        const uint64_t v = (uint64_t)(list_id(a.seen, row * a.ld_seen + i, a.ids64 & 1) - c0);
        if (v < (uint64_t)len) atomicAdd(&count[v], 1u);
      }
    }
    if (a.bias_ids) {
      for (int64_t i = threadIdx.x; i < a.n_bias; i += kThreads) {
        const uint64_t v = (uint64_t)(list_id(a.bias_ids, row * a.ld_bias + i, a.ids64 & 2) - c0);
        if (v < (uint64_t)len) atomicMax(&slot[v], (uint32_t)i + 1u);
      }
    }
    __syncthreads();
  }
  const float rep = a.repetition ? a.repetition[row] : a.repetition_all;
  const float pre = a.presence ? a.presence[row] : a.presence_all;
  const float fre = a.frequency ? a.frequency[row] : a.frequency_all;
  const T* src = (const T*)a.scores + row * a.ld_scores + c0;
  T* dst = (T*)a.out + row * a.ld_out + c0;
  const uint32_t* mask = a.mask ? a.mask + row * a.ld_mask + (c0 >> 5) : nullptr;
  typedef typename Vec8<T>::type V;
  auto one = [&](float x, int i) {
    if (a.seen) {
      const uint32_t c = count[i];
      if (c) x = (x > 0.f ? x / rep : x * rep) - (fre * (float)c + pre);
    }
    if (a.bias_ids) {
      const uint32_t s = slot[i];
      if (s) x += a.bias[row * a.ld_bias + (s - 1)];
    }
    return x;
  };
  for (int i = threadIdx.x * kVec; i < len; i += kThreads * kVec) {
    const uint32_t bits = mask ? mask[i >> 5] >> (i & 31) : 0xFFu;
    if (i + kVec <= len) {
      V v = *(const V*)(src + i);
#pragma unroll
      for (int j = 0; j < kVec; ++j) v[j] = (bits >> j) & 1 ? (T)one((float)v[j], i + j) : (T)-__builtin_inff();
      *(V*)(dst + i) = v;
    } else {
      for (int j = 0; i + j < len; ++j)
        dst[i + j] = (bits >> j) & 1 ? (T)one((float)src[i + j], i + j) : (T)-__builtin_inff();
    }
  }
}

int check(const bb_adjust* a) {
  const char* fn = "bb_adjust_scores: ";
  auto bad = [&](const char* why) { return abi_fail(BB_E_ARG, std::string(fn) + why); };
  if (!a) return bad("null arguments");
  if (a->dtype != BB_F32 && a->dtype != BB_BF16 && a->dtype != BB_F16) return bad("dtype must be BB_F32, BB_BF16 or BB_F16");
  if (a->B < 0 || a->n < 0) return bad("negative size");
  if (a->n > 0x7FFFFFFF || a->n_seen > 0x7FFFFFFF || a->n_bias > 0x7FFFFFFF) return bad("n and the lists are below 2^31");
  if (a->B == 0 || a->n == 0) return BB_OK;
  if (!a->scores || !a->out) return bad("null scores or out");
  if (a->ld_scores < a->n || a->ld_out < a->n) return bad("rows overlap (ld < n)");
  const uintptr_t es = a->dtype == BB_F32 ? 4 : 2;
  const uintptr_t s0 = (uintptr_t)a->scores, o0 = (uintptr_t)a->out;
  if (s0 % es || o0 % es) return bad("scores or out is not aligned to its type");
  if (a->B > 0x7FFFFFFF) return bad("too many rows for one call");
  const uint64_t s_bytes = ((uint64_t)(a->B - 1) * a->ld_scores + a->n) * es;
  const uint64_t o_bytes = ((uint64_t)(a->B - 1) * a->ld_out + a->n) * es;
  if (overlap(a->scores, s_bytes, a->out, o_bytes) && !(s0 == o0 && a->ld_scores == a->ld_out))
    return bad("out overlaps scores without being the same rows");
  if (a->n_seen < 0 || a->n_bias < 0) return bad("negative list length");
  if (a->n_seen > 0 && !a->seen) return bad("n_seen without seen");
  if (a->n_bias > 0 && (!a->bias_ids || !a->bias)) return bad("n_bias without bias_ids and bias");
  if (a->seen && a->ld_seen != 0 && a->ld_seen < a->n_seen) return bad("ld_seen < n_seen");
  if (a->bias_ids && a->ld_bias != 0 && a->ld_bias < a->n_bias) return bad("ld_bias < n_bias");
  if (a->mask && a->ld_mask != 0 && a->ld_mask < (a->n + 31) / 32) return bad("ld_mask < ceil(n/32)");
  const uintptr_t is = a->ids64 & 1 ? 8 : 4, ib = a->ids64 & 2 ? 8 : 4;
  if ((uintptr_t)a->seen % is || (uintptr_t)a->bias_ids % ib || (uintptr_t)a->seen_len % 4 || (uintptr_t)a->bias % 4 ||
      (uintptr_t)a->mask % 4 || (uintptr_t)a->repetition % 4 || (uintptr_t)a->presence % 4 || (uintptr_t)a->frequency % 4)
    return bad("a list, mask or parameter is not aligned to its type");
  return BB_OK;
}

}  // namespace
}  // namespace bb

extern "C" int bb_adjust_scores(int32_t device, const bb_adjust* args, void* stream) {
  using namespace bb;
  return abi_call("bb_adjust_scores", [&]() -> int {
    int rc = check(args);
    if (rc || args->B == 0 || args->n == 0) return rc;
    bb_adjust a = *args;
    if (a.n_seen == 0) a.seen = nullptr;
    if (a.n_bias == 0) a.bias_ids = nullptr;
    const int64_t n_chunks = (a.n + kChunk - 1) / kChunk;
    // a launch holds less than 2^32 threads
    if (a.B > (int64_t)(0xFFFFFFFFu / kThreads) / n_chunks)
      return abi_fail(BB_E_ARG, "bb_adjust_scores: too many rows for one call");
    CallDevice dev;
    if ((rc = dev.enter(device, "bb_adjust_scores"))) return rc;
    const uint32_t lds = ((a.seen ? kChunk : 0) + (a.bias_ids ? kChunk : 0)) * 4;
    const dim3 grid((uint32_t)(a.B * n_chunks));
    auto go = [&](auto kernel) {
      return abi_launch("bb_adjust_scores", kernel, grid, dim3(kThreads), lds, (hipStream_t)stream, a, (int)n_chunks);
    };
    if (a.dtype == BB_F32) return go(adjust_kernel<float>);
    if (a.dtype == BB_BF16) return go(adjust_kernel<__bf16>);
    return go(adjust_kernel<_Float16>);
  });
}
