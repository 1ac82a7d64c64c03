// Global norm over many gradient tensors, and clipping by it.
//
//   s = sqrt(sum over tensors of sum g^2),  g' = g min(1, max_norm / (s + eps))
//
// Two launches whatever the number of tensors (up to kGradTensors a launch): the tensors' addresses
// and sizes travel as kernel parameters, so nothing is uploaded and a captured graph replays the call.
// The tensors are cut into equal chunks that the blocks take in a fixed order; each block writes one
// 64-bit partial sum, and every block of the second launch adds all of them up for itself in the same
// order, so the result does not depend on which block ran first and no counter has to be reset.
// Squares are added in 64 bits: a norm neither overflows nor vanishes before its own value does.
//
// What bounds it: memory; the gradients are read twice and written once. The second launch walks the
// chunks backwards, from the ones that the first read last (1% on a list of 247 MB; evict-last and streaming
// cache hints gave no more: B200 writes at 3.8 TB/s at most, and that, not the second read, is what the
// second launch waits for).
#pragma once

#include "distill_common.cuh"
#include "orda_b200_student.h"

namespace orda {

constexpr int kGradThreads = 256;

template <int N>
struct GradTable {
  const void* src[N];
  void* dst[N];
  int64_t numel[N];
  int32_t first_chunk[N + 1];  // [count] = number of chunks
  uint8_t dtype[N];
  int32_t count;
  int32_t chunk;               // elements per chunk, a multiple of 8 * kGradThreads
};

// Tensor that holds chunk c: the last one whose first chunk is not behind c (empty tensors have none).
template <int N>
__device__ __forceinline__ int tensor_of(const GradTable<N>& g, int c) {
  int lo = 0, hi = g.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (g.first_chunk[mid] <= c) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ double square(float x) { return static_cast<double>(x) * static_cast<double>(x); }

__device__ __forceinline__ double block_sum(double v, double* shared) {
  for (int o = 16; o > 0; o /= 2) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if (threadIdx.x % 32 == 0) shared[threadIdx.x / 32] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int k = 0; k < kGradThreads / 32; ++k) v += shared[k];
  return v;
}

// 16 bytes of T as floats
template <typename T>
__device__ __forceinline__ void unpack16(const uint4& u, float (&v)[16 / sizeof(T)]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) unpack2<T>(w[i], v[2 * i], v[2 * i + 1]);
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack16(const float (&v)[16 / sizeof(T)]) {
  if constexpr (sizeof(T) == 4)
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  else
    return make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
}

// Sum of squares of one 16-byte vector. 16-bit types: the eight squares are formed and added in fp32 (exact
// products) and converted once, since converting every value to fp64 bounds the kernel by the conversion
// pipe (393 us against 364 for 1.2e9 bf16 values); a sum near either end of fp32's range is taken again in fp64.
template <typename T>
__device__ __forceinline__ double vector_squares(const uint4& u) {
  constexpr int V = 16 / sizeof(T);
  float v[V];
  unpack16<T>(u, v);
  if constexpr (sizeof(T) == 2) {
    float a = v[0] * v[0], b = v[1] * v[1];
#pragma unroll
    for (int e = 2; e < V; e += 2) {
      a = fmaf(v[e], v[e], a);
      b = fmaf(v[e + 1], v[e + 1], b);
    }
    a += b;
    if (a > 1e-27f && a < 1e36f) return static_cast<double>(a);
  }
  double s = 0.0;
#pragma unroll
  for (int e = 0; e < V; ++e) s += square(v[e]);
  return s;
}

template <typename T>
__device__ __forceinline__ double chunk_squares(const T* p, int64_t n) {
  constexpr int V = 16 / sizeof(T);
  double acc[2] = {0.0, 0.0};
  int64_t done = 0;
  if ((reinterpret_cast<uintptr_t>(p) & 15u) == 0) {
    const int64_t vecs = n / V;
    const uint4* q = reinterpret_cast<const uint4*>(p);
    int64_t i = threadIdx.x;
    for (; i + 3 * kGradThreads < vecs; i += 4 * kGradThreads) {
      uint4 u[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) u[k] = __ldg(q + i + k * kGradThreads);
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[k & 1] += vector_squares<T>(u[k]);
    }
    for (; i < vecs; i += kGradThreads) acc[0] += vector_squares<T>(__ldg(q + i));
    done = vecs * V;
  }
  for (int64_t i = done + threadIdx.x; i < n; i += kGradThreads) acc[0] += square(Conv<T>::to_f(p[i]));
  return acc[0] + acc[1];
}

template <typename T>
__device__ __forceinline__ void chunk_scale(const T* p, T* d, int64_t n, float c, float c2) {
  constexpr int V = 16 / sizeof(T);
  int64_t done = 0;
  if (((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(d)) & 15u) == 0) {
    const int64_t vecs = n / V;
    const uint4* q = reinterpret_cast<const uint4*>(p);
    uint4* o = reinterpret_cast<uint4*>(d);
    int64_t i = threadIdx.x;
    for (; i + 3 * kGradThreads < vecs; i += 4 * kGradThreads) {
      uint4 u[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) u[k] = q[i + k * kGradThreads];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float v[V];
        unpack16<T>(u[k], v);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = v[e] * c * c2;
        o[i + k * kGradThreads] = pack16<T>(v);
      }
    }
    for (; i < vecs; i += kGradThreads) {
      float v[V];
      unpack16<T>(q[i], v);
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = v[e] * c * c2;
      o[i] = pack16<T>(v);
    }
    done = vecs * V;
  }
  for (int64_t i = done + threadIdx.x; i < n; i += kGradThreads) d[i] = Conv<T>::from_f(Conv<T>::to_f(p[i]) * c * c2);
}

template <int N>
__global__ void __launch_bounds__(kGradThreads) grad_squares_kernel(const __grid_constant__ GradTable<N> g,
                                                                    double* partial) {
  __shared__ double shared[kGradThreads / 32];
  double acc = 0.0;
  const int chunks = g.first_chunk[g.count];
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int t = tensor_of(g, c);
    const int64_t at = static_cast<int64_t>(c - g.first_chunk[t]) * g.chunk;
    const int64_t n = min(static_cast<int64_t>(g.chunk), g.numel[t] - at);
    if (g.dtype[t] == ORDA_F32) acc += chunk_squares(static_cast<const float*>(g.src[t]) + at, n);
    else if (g.dtype[t] == ORDA_F16) acc += chunk_squares(static_cast<const __half*>(g.src[t]) + at, n);
    else acc += chunk_squares(static_cast<const __nv_bfloat16*>(g.src[t]) + at, n);
  }
  acc = block_sum(acc, shared);
  if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

// Every block's own sum of all partial sums: the norm.
__device__ __forceinline__ double norm_of(const double* partial, int parts, double* shared) {
  double v = 0.0;
  for (int i = threadIdx.x; i < parts; i += kGradThreads) v += partial[i];
  return sqrt(block_sum(v, shared));
}

static __global__ void __launch_bounds__(kGradThreads) grad_norm_kernel(const double* partial, int parts, float* norm) {
  __shared__ double shared[kGradThreads / 32];
  const double s = norm_of(partial, parts, shared);
  if (threadIdx.x == 0) *norm = static_cast<float>(s);
}

template <int N>
__global__ void __launch_bounds__(kGradThreads) grad_scale_kernel(const __grid_constant__ GradTable<N> g,
                                                                  const double* partial, int parts, double max_norm,
                                                                  double eps, float* norm) {
  __shared__ double shared[kGradThreads / 32];
  const double s = norm_of(partial, parts, shared);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(s);
  const double ratio = max_norm / (s + eps);
  // below fp32's normal range the factor would lose bits that the values have: it is taken in two steps
  const bool tiny = ratio < 0x1p-126;
  const float factor = ratio >= 1.0 ? 1.f : static_cast<float>(tiny ? ratio * 0x1p64 : ratio);  // NaN stays NaN
  const float rest = tiny ? 0x1p-64f : 1.f;
  const int chunks = g.first_chunk[g.count];
  for (int c = chunks - 1 - static_cast<int>(blockIdx.x); c >= 0; c -= static_cast<int>(gridDim.x)) {
    const int t = tensor_of(g, c);
    if (factor == 1.f && g.dst[t] == g.src[t]) continue;  // in place and unchanged
    const int64_t at = static_cast<int64_t>(c - g.first_chunk[t]) * g.chunk;
    const int64_t n = min(static_cast<int64_t>(g.chunk), g.numel[t] - at);
    if (g.dtype[t] == ORDA_F32)
      chunk_scale(static_cast<const float*>(g.src[t]) + at, static_cast<float*>(g.dst[t]) + at, n, factor, rest);
    else if (g.dtype[t] == ORDA_F16)
      chunk_scale(static_cast<const __half*>(g.src[t]) + at, static_cast<__half*>(g.dst[t]) + at, n, factor, rest);
    else
      chunk_scale(static_cast<const __nv_bfloat16*>(g.src[t]) + at, static_cast<__nv_bfloat16*>(g.dst[t]) + at, n,
                  factor, rest);
  }
}

}  // namespace orda
