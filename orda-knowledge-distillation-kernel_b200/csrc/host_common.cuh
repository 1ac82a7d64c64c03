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

inline int num_sms() {
  int dev = 0, n = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n > 0 ? n : 148;
}

inline size_t align256(size_t x) { return (x + 255) & ~size_t(255); }
inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline size_t esize(int dtype) { return dtype == ORDA_F32 ? 4 : 2; }
inline int launch_status() { return cudaPeekAtLastError() == cudaSuccess ? ORDA_OK : ORDA_ERR_CUDA; }

}  // namespace orda
