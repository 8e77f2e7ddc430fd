// abi.h — what the entry points outside api.hip share: the error state behind bb_last_error,
// the device of a call, and launches whose own status is returned.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

#include "../../include/brickrec.h"

namespace bb {

// Sets this thread's bb_last_error() message (api.hip) and returns `code`.
int abi_fail(int code, const std::string& msg);

// No C++ exception leaves an entry point.
template <typename F>
inline int abi_call(const char* fn, F&& body) noexcept {
  try {
    return body();
  } catch (...) {
    try {
      return abi_fail(BB_E_NOMEM, std::string(fn) + ": out of host memory");
    } catch (...) {
      return BB_E_NOMEM;
    }
  }
}

// Whether [a, a + na) and [b, b + nb) share a byte.
inline bool overlap(const void* a, uint64_t na, const void* b, uint64_t nb) {
  return na && nb && (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na;
}

// The device of a call for its duration (-1 = the current one).
struct CallDevice {
  int prev = -1;
  bool moved = false;
  int enter(int dev, const char* fn) {
    hipError_t e = hipGetDevice(&prev);
    if (e == hipSuccess && dev >= 0 && dev != prev) {
      e = hipSetDevice(dev);
      moved = e == hipSuccess;
    }
    return e == hipSuccess ? BB_OK : abi_fail(BB_E_HIP, std::string(fn) + ": device " + std::to_string(dev) + ": " + hipGetErrorString(e));
  }
  ~CallDevice() {
    if (moved) (void)hipSetDevice(prev);
  }
};

template <typename T>
struct AsIs {
  using type = T;
};
// One launch; the status is the launch's own, not an older call's.
template <typename... KArgs>
inline int abi_launch(const char* fn, void (*kernel)(KArgs...), dim3 grid, dim3 block, uint32_t lds, hipStream_t s,
                      typename AsIs<KArgs>::type... args) {
  void* argv[] = {(void*)&args...};
  const hipError_t e = hipLaunchKernel((const void*)kernel, grid, block, argv, lds, s);
  return e == hipSuccess ? BB_OK : abi_fail(BB_E_HIP, std::string(fn) + ": launch: " + hipGetErrorString(e));
}

}  // namespace bb
