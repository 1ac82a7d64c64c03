// Host-side helpers shared by the translation units of the library.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <atomic>

#include "orda_b200.h"

namespace orda {

// kernels launched by this library in this process (orda_kernel_launches)
inline std::atomic<uint64_t> g_launches{0};
inline void count_launch(uint64_t n = 1) { g_launches.fetch_add(n, std::memory_order_relaxed); }

// SMs of the current device (asked once per device: a launch of a few microseconds calls this twice).
inline int num_sms() {
  static std::atomic<int> known[64];
  int dev = 0, n = 0;
  cudaGetDevice(&dev);
  const bool slot = dev >= 0 && dev < 64;
  if (slot && (n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  if (n <= 0) return 148;
  if (slot) known[dev].store(n, std::memory_order_relaxed);
  return n;
}

inline size_t align256(size_t x) { return (x + 255) & ~size_t(255); }
inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline size_t esize(int dtype) { return dtype == ORDA_F32 ? 4 : 2; }
// Result of the launches since the last check. It takes the error with it: left pending, a failed launch would
// be reported again by the thread's next call, whose own launches went well.
inline int launch_status() { return cudaGetLastError() == cudaSuccess ? ORDA_OK : ORDA_ERR_CUDA; }

}  // namespace orda
