// adjust.hip — penalties for ids seen already, sparse biases and a bit mask on dense scores
// (bb_adjust_scores).
//
// One pass over the scores, bound by moving them.  A workgroup takes one chunk of one row.  Its scores
// and mask bits are loaded first; while they are on their way, the row's lists are read (from the L2: every
// chunk of a row reads them again, so long lists get larger chunks) and what concerns the chunk is
// kept in LDS, one word a score: the position of the last bias entry of the id in the high half,
// how often it was seen in the low half.  Integer maxima and sums, so their order does not matter.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

#include "abi.h"

namespace bb {
namespace {

constexpr int kVec = 8;  // scores per thread: 16 bytes of a 16-bit type, a byte of the mask

template <typename T, int N>
struct VecOf {
  typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};

// A row's list of ids, 4 at a time to a thread; the first 4 are loaded when it is made, so that their
// latency passes beside that of the scores.
template <int THREADS, typename Id>
struct List {
  typedef typename VecOf<Id, 4>::type V;
  const Id* ids;
  int n;
  V first;
  __device__ __forceinline__ List(const void* p, int64_t at, int n_) : ids((const Id*)p + at), n(n_) {
    if ((int)threadIdx.x * 4 + 4 <= n) first = *(const V*)(ids + threadIdx.x * 4);
  }
  // f(entry, id) for the first `m` <= n entries
  template <typename F>
  __device__ __forceinline__ void each(int m, F&& f) const {
    for (int i = threadIdx.x * 4; i < m; i += THREADS * 4) {
      if (i + 4 <= n) {
        const V v = i < THREADS * 4 ? first : *(const V*)(ids + i);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (i + j < m) f(i + j, (int64_t)v[j]);
      } else {
        for (int j = i; j < m; ++j) f(j, (int64_t)ids[j]);
      }
    }
  }
};

// SPLIT: lists of 2^16 entries or more, whose counts and positions take a word each.
template <typename T, typename Id, int THREADS, bool SPLIT>
__global__ __launch_bounds__(THREADS) void adjust_kernel(bb_adjust a, int n_chunks) {
  constexpr int kChunk = THREADS * kVec;
  __shared__ __attribute__((aligned(16))) uint32_t lds[kChunk * (SPLIT ? 2 : 1)];
  const int64_t row = blockIdx.x / n_chunks;
  const int64_t c0 = (int64_t)(blockIdx.x % n_chunks) * kChunk;
  const int len = (int)(a.n - c0 < kChunk ? a.n - c0 : kChunk);
  const T* src = (const T*)a.scores + row * a.ld_scores + c0;
  T* dst = (T*)a.out + row * a.ld_out + c0;
  const uint32_t* mask = a.mask ? a.mask + row * a.ld_mask + (c0 >> 5) : nullptr;
  typedef typename VecOf<T, kVec>::type V;
  typedef uint32_t W __attribute__((ext_vector_type(4)));
  const int i = threadIdx.x * kVec;  // this thread's 8 scores of the chunk
  V v;
  uint32_t bits = 0xFFu;
  if (i < len && mask) bits = mask[i >> 5] >> (i & 31);
  if (i + kVec <= len) v = *(const V*)(src + i);
  const float rep = a.repetition ? a.repetition[row] : a.repetition_all;
  const float pre = a.presence ? a.presence[row] : a.presence_all;
  const float fre = a.frequency ? a.frequency[row] : a.frequency_all;
  const bool lists = a.seen || a.bias_ids;
  if (lists) {
    const List<THREADS, Id> seen(a.seen, row * a.ld_seen, a.seen ? (int)a.n_seen : 0);
    const List<THREADS, Id> biased(a.bias_ids, row * a.ld_bias, a.bias_ids ? (int)a.n_bias : 0);
    int n_seen = seen.n;
    if (a.seen && a.seen_len) {
      const int l = a.seen_len[row];
      n_seen = l < 0 ? 0 : l < n_seen ? l : n_seen;
    }
#pragma unroll
    for (int z = 0; z < kChunk * (SPLIT ? 2 : 1) / 4; z += THREADS) *(W*)(lds + (z + threadIdx.x) * 4) = W{0, 0, 0, 0};
    __syncthreads();
    uint32_t* slot = SPLIT ? lds + kChunk : lds;
    if (a.bias_ids) {
      biased.each(biased.n, [&](int e, int64_t id) {
        const uint64_t at = (uint64_t)id - (uint64_t)c0;  // (ids below the chunk wrap to far above it)
        if (at < (uint64_t)len) atomicMax(&slot[at], SPLIT ? (uint32_t)e + 1u : ((uint32_t)e + 1u) << 16);
      });
      if (!SPLIT && a.seen) __syncthreads();  // (the maxima are over words whose counts are still 0)
    }
    seen.each(n_seen, [&](int, int64_t id) {
      const uint64_t at = (uint64_t)id - (uint64_t)c0;
      if (at < (uint64_t)len) atomicAdd(&lds[at], 1u);
    });
    __syncthreads();
  }
  const float* bias = a.bias_ids ? a.bias + row * a.ld_bias : nullptr;
  auto one = [&](float x, uint32_t count, uint32_t slot) {
    if (count) x = (x > 0.f ? x / rep : x * rep) - (fre * (float)count + pre);
    if (slot) x += bias[slot - 1];
    return x;
  };
  auto count_of = [&](uint32_t w) { return SPLIT ? w : w & 0xFFFFu; };
  if (i + kVec <= len) {
    if (lists) {
      uint32_t w[kVec], t[kVec];
#pragma unroll
      for (int j = 0; j < kVec; j += 4) {
        *(W*)&w[j] = *(const W*)(lds + i + j);
        if constexpr (SPLIT) *(W*)&t[j] = *(const W*)(lds + kChunk + i + j);
      }
      uint32_t any = 0;
#pragma unroll
      for (int j = 0; j < kVec; ++j) any |= SPLIT ? w[j] | t[j] : w[j];
      if (any) {  // (most groups of 8 hold no listed id)
#pragma unroll
        for (int j = 0; j < kVec; ++j) v[j] = (T)one((float)v[j], count_of(w[j]), SPLIT ? t[j] : w[j] >> 16);
      }
    }
#pragma unroll
    for (int j = 0; j < kVec; ++j) v[j] = (bits >> j) & 1 ? v[j] : (T)-__builtin_inff();
    *(V*)(dst + i) = v;
  } else {
    for (int j = 0; i + j < len; ++j) {
      float x = (float)src[i + j];
      if (lists) x = one(x, count_of(lds[i + j]), SPLIT ? lds[kChunk + i + j] : lds[i + j] >> 16);
      dst[i + j] = (bits >> j) & 1 ? (T)x : (T)-__builtin_inff();
    }
  }
}

int check(const bb_adjust* a) {
  const char* fn = "bb_adjust_scores: ";
  auto bad = [&](const char* why) { return abi_fail(BB_E_ARG, std::string(fn) + why); };
  if (!a) return bad("null arguments");
  if (a->dtype != BB_F32 && a->dtype != BB_BF16 && a->dtype != BB_F16) return bad("dtype must be BB_F32, BB_BF16 or BB_F16");
  if (a->B < 0 || a->n < 0) return bad("negative size");
  if (a->n > 0x7FFFFFFF || a->n_seen >= 1 << 30 || a->n_bias >= 1 << 30) return bad("n is below 2^31, the lists below 2^30");
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
  const uintptr_t ib = a->ids64 ? 8 : 4;
  if ((uintptr_t)a->seen % ib || (uintptr_t)a->bias_ids % ib || (uintptr_t)a->seen_len % 4 || (uintptr_t)a->bias % 4 ||
      (uintptr_t)a->mask % 4 || (uintptr_t)a->repetition % 4 || (uintptr_t)a->presence % 4 || (uintptr_t)a->frequency % 4)
    return bad("a list, mask or parameter is not aligned to its type");
  // what other workgroups may still read
  auto meets = [&](const void* p, int64_t n, int64_t ld, uint64_t size) {
    return p && n > 0 && overlap(p, ((uint64_t)(a->B - 1) * ld + n) * size, a->out, o_bytes);
  };
  if (meets(a->seen, a->n_seen, a->ld_seen, ib) || meets(a->bias_ids, a->n_bias, a->ld_bias, ib) ||
      meets(a->bias, a->n_bias, a->ld_bias, 4) || meets(a->mask, (a->n + 31) / 32, a->ld_mask, 4) ||
      meets(a->seen_len, 1, 1, 4) || meets(a->repetition, 1, 1, 4) || meets(a->presence, 1, 1, 4) ||
      meets(a->frequency, 1, 1, 4))
    return bad("out overlaps a list, the mask or a parameter");
  return BB_OK;
}

template <typename T, typename Id, int THREADS, bool SPLIT>
int launch(const bb_adjust& a, void* stream) {
  constexpr int kChunk = THREADS * kVec;
  const int64_t n_chunks = (a.n + kChunk - 1) / kChunk;
  // a launch holds less than 2^32 threads
  if (a.B > (int64_t)(0xFFFFFFFFu / THREADS) / n_chunks) return abi_fail(BB_E_ARG, "bb_adjust_scores: too many rows for one call");
  return abi_launch("bb_adjust_scores", adjust_kernel<T, Id, THREADS, SPLIT>, dim3((uint32_t)(a.B * n_chunks)),
                    dim3(THREADS), 0, (hipStream_t)stream, a, (int)n_chunks);
}

template <typename T, typename Id>
int launch_type(const bb_adjust& a, void* stream) {
  if (a.n_seen >= 1 << 16 || a.n_bias >= 1 << 16) return launch<T, Id, 1024, true>(a, stream);
  // Longer lists are read by fewer, larger workgroups: 64 rows of 131,072 bf16 with 4,096 ids each take 15.8 us with
  // 256 threads and 13.3 with 1024; 256 rows of 25,216 f32 with 200 ids 12.3 and 14.9 (copying those
  // scores alone: 7.1 and 11.0 us at the 4.7 TB/s of a large copy).  One row of 25,216: 3.7 us.
  if (a.n_seen + a.n_bias > 1024) return launch<T, Id, 1024, false>(a, stream);
  return launch<T, Id, 256, false>(a, stream);
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
    CallDevice dev;
    if ((rc = dev.enter(device, "bb_adjust_scores"))) return rc;
    auto go = [&](auto id) {
      using Id = decltype(id);
      return a.dtype == BB_F32 ? launch_type<float, Id>(a, stream)
             : a.dtype == BB_BF16 ? launch_type<__bf16, Id>(a, stream)
                                  : launch_type<_Float16, Id>(a, stream);
    };
    return a.ids64 ? go(int64_t{}) : go(int32_t{});
  });
}
