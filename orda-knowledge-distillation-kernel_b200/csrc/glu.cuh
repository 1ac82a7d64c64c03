// Gated feed-forward block for a few rows, and the pointwise kernels of the block.
//
//   h = act(g) u,  g = x Wg^T,  u = x Wu^T
//   dg = dh u act'(g),  du = dh act(g)
//
// Many rows run on the pair GEMMs (gemm_tc2w.cuh, gemm_tc2.cuh, EPI_GLU), up to 128 on glu_swap.cuh. With at
// most 8 rows the two weights are all that has to be read, so glu_rows_kernel streams them once, straight from memory into the fragments
// of mma.sync (m16n8k16): 16 features of each weight a block, the block's 8 warps share out K, the
// partial sums meet in shared memory in a fixed order. A lane's 16-byte load holds 8 consecutive k of one
// weight row; which of them an instruction takes as its k = 0 .. 15 is free as long as x is permuted
// alike, so lane t of a quad feeds k 8t .. 8t+3 to one instruction and 8t+4 .. 8t+7 to the next and
// nothing is shuffled or staged.
//
// What bounds it: reading the weights. One row, 4096 -> 11264 in bf16 takes 34.9 us, 5.3 TB/s (80% of a copy);
// 4 warps a block took 39, half the loads in flight 38. From 9 rows on the tensor-memory kernel is as
// fast, and with more fragments of x this one fell behind (32 rows: 62 us against 39).
#pragma once

#include <type_traits>

#include "distill_common.cuh"
#include "glu_math.cuh"
#include "orda_b200_student.h"

namespace orda {

constexpr int kGluWarps = 8;
constexpr int kGluFeatures = 16;  // features of a block
constexpr int kGluK = 32;         // k elements of one 16-byte load per lane
constexpr int kGluUnroll = 4;     // loads of each row in flight: 128 k a step

struct GluRowsParams {
  const void *x, *gate, *up;
  void *h, *pre_gate, *pre_up;
  int64_t ld_x, ld_gate, ld_up, ld_h, ld_pre;
  int64_t ffn;
  int32_t rows, hidden, act;
};

template <typename T>
__device__ __forceinline__ void mma_16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                            uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes that this kernel reads once: no reuse in L1
__device__ __forceinline__ uint4 load_stream(const void* p) {
  uint4 u;
  asm volatile("ld.global.nc.L1::no_allocate.L2::128B.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
               : "l"(p));
  return u;
}

// At most 8 rows: one n = 8 fragment of x.
template <typename T>
__global__ void __launch_bounds__(32 * kGluWarps) glu_rows_kernel(const __grid_constant__ GluRowsParams p) {
  __shared__ float part[kGluWarps][2][kGluFeatures][8 + 1];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int r = lane / 4, q = lane % 4;
  const int64_t f0 = static_cast<int64_t>(blockIdx.x) * kGluFeatures;
  // rows r and r + 8 of the block's features in each weight; features behind the last read row 0's and
  // are dropped
  const int64_t fa = f0 + r < p.ffn ? f0 + r : 0, fb = f0 + r + 8 < p.ffn ? f0 + r + 8 : 0;
  const T* g0 = static_cast<const T*>(p.gate) + fa * p.ld_gate;
  const T* g1 = static_cast<const T*>(p.gate) + fb * p.ld_gate;
  const T* u0 = static_cast<const T*>(p.up) + fa * p.ld_up;
  const T* u1 = static_cast<const T*>(p.up) + fb * p.ld_up;
  float cg[4] = {}, cu[4] = {};
  const uint4 zero = make_uint4(0, 0, 0, 0);
  for (int k0 = warp * kGluK * kGluUnroll; k0 < p.hidden; k0 += kGluWarps * kGluK * kGluUnroll) {
    uint4 w[kGluUnroll][4];
#pragma unroll
    for (int j = 0; j < kGluUnroll; ++j) {
      const int k = k0 + j * kGluK + q * 8;
      const bool on = k < p.hidden;  // hidden is a multiple of 8
      w[j][0] = on ? load_stream(g0 + k) : zero;
      w[j][1] = on ? load_stream(g1 + k) : zero;
      w[j][2] = on ? load_stream(u0 + k) : zero;
      w[j][3] = on ? load_stream(u1 + k) : zero;
    }
#pragma unroll
    for (int j = 0; j < kGluUnroll; ++j) {
      const int k = k0 + j * kGluK + q * 8;
      uint4 x = zero;
      if (r < p.rows && k < p.hidden)
        x = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.x) + r * p.ld_x + k));
      mma_16x8x16<T>(cg, w[j][0].x, w[j][1].x, w[j][0].y, w[j][1].y, x.x, x.y);
      mma_16x8x16<T>(cg, w[j][0].z, w[j][1].z, w[j][0].w, w[j][1].w, x.z, x.w);
      mma_16x8x16<T>(cu, w[j][2].x, w[j][3].x, w[j][2].y, w[j][3].y, x.x, x.y);
      mma_16x8x16<T>(cu, w[j][2].z, w[j][3].z, w[j][2].w, w[j][3].w, x.z, x.w);
    }
  }
  // accumulator element e of a lane: feature r (+ 8 for e >= 2), row 2 q + (e & 1)
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    part[warp][0][r + (e >> 1) * 8][2 * q + (e & 1)] = cg[e];
    part[warp][1][r + (e >> 1) * 8][2 * q + (e & 1)] = cu[e];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kGluFeatures * p.rows; i += 32 * kGluWarps) {
    const int f = i % kGluFeatures, row = i / kGluFeatures;
    if (f0 + f >= p.ffn) continue;
    float g = 0.f, u = 0.f;
#pragma unroll
    for (int k = 0; k < kGluWarps; ++k) {
      g += part[k][0][f][row];
      u += part[k][1][f][row];
    }
    float a = 0.f, d;
    with_act(p.act, [&](auto tag) { glu_act<decltype(tag)::kAct, false>(g, a, d); });
    static_cast<T*>(p.h)[row * p.ld_h + f0 + f] = Conv<T>::from_f(a * u);
    if (p.pre_gate) {
      static_cast<T*>(p.pre_gate)[row * p.ld_pre + f0 + f] = Conv<T>::from_f(g);
      static_cast<T*>(p.pre_up)[row * p.ld_pre + f0 + f] = Conv<T>::from_f(u);
    }
  }
}

// h = act(g) u of the fp32 path. Rows of `cols` values, row stride ld of g and u, ld_h of h.
static __global__ void __launch_bounds__(256) glu_act_kernel(const float* g, const float* u, float* h, int64_t rows,
                                                             int64_t cols, int64_t ld, int64_t ld_h, int act) {
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < rows * cols;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t at = i / cols * ld + i % cols;
    float a = 0.f, d;
    with_act(act, [&](auto tag) { glu_act<decltype(tag)::kAct, true>(g[at], a, d); });
    h[i / cols * ld_h + i % cols] = a * u[at];
  }
}

// What a product is formed from again: rows of `hidden` elements, a multiple of 8, 16-byte aligned.
struct GluSources {
  const void *x, *gate, *up;
  int64_t ld_x, ld_gate, ld_up, hidden;
};

// sum a[k] b[k] in fp32
static __device__ __noinline__ float dot_f16(const __half* a, const __half* b, int64_t n) {
  float acc[2] = {0.f, 0.f};
  for (int64_t k = 0; k < n; k += 8) {
    const uint4 ua = __ldg(reinterpret_cast<const uint4*>(a + k)), ub = __ldg(reinterpret_cast<const uint4*>(b + k));
    const uint32_t wa[4] = {ua.x, ua.y, ua.z, ua.w}, wb[4] = {ub.x, ub.y, ub.z, ub.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float a0, a1, b0, b1;
      unpack2<__half>(wa[j], a0, a1);
      unpack2<__half>(wb[j], b0, b1);
      acc[0] = fmaf(a0, b0, acc[0]);
      acc[1] = fmaf(a1, b1, acc[1]);
    }
  }
  return acc[0] + acc[1];
}

// dg and du into the two halves of `out`, rows of 2 * cols_pad: columns [0, cols_pad) dg, the rest du.
// g, u and out 16-byte aligned, cols_pad and ld (the row stride of g and u) multiples of 8; dh (row stride
// ld_dh) any, read element by element unless dh_vec. The columns behind `cols` (the padding) are set to
// zero. One 8-element vector per thread and step; memory-bound (three reads, two writes).
//
// fp16: h comes from fp32 products, and may be finite where a product is beyond 65504 and was saved as an
// infinity (silu(-1e5) is 0). Read as one, it would give inf * 0 = NaN for a gradient that is 0, so a product
// that is saved as an infinity is formed again in fp32 (and is infinite again if x or a weight is).
template <typename T>
__global__ void __launch_bounds__(256) glu_grad_kernel(const T* __restrict__ dh, int64_t ld_dh, int dh_vec,
                                                       const T* __restrict__ g, const T* __restrict__ u,
                                                       T* __restrict__ out, int64_t rows, int64_t cols,
                                                       int64_t cols_pad, int64_t ld, int act, int32_t* status,
                                                       const GluSources src) {
  if (status && blockIdx.x == 0 && threadIdx.x == 0) *status = 0;  // for the gradient GEMMs that follow
  const int64_t vecs = cols_pad / 8, total = rows * vecs;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t row = i / vecs, c = (i - row * vecs) * 8;
    const int64_t at = row * ld + c;
    float vd[8], vg[8], vu[8];
    [[maybe_unused]] float largest = 0.f;
    constexpr int Q = sizeof(T) / 2;
#pragma unroll
    for (int k = 0; k < Q; ++k) {
      uint4 a = make_uint4(0, 0, 0, 0);
      if (dh_vec) a = __ldcs(reinterpret_cast<const uint4*>(dh + row * ld_dh + c) + k);
      const uint4 b = __ldcs(reinterpret_cast<const uint4*>(g + at) + k);
      const uint4 e = __ldcs(reinterpret_cast<const uint4*>(u + at) + k);
      const uint32_t wa[4] = {a.x, a.y, a.z, a.w}, wb[4] = {b.x, b.y, b.z, b.w}, we[4] = {e.x, e.y, e.z, e.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 4) {
          vd[k * 4 + j] = __uint_as_float(wa[j]);
          vg[k * 4 + j] = __uint_as_float(wb[j]);
          vu[k * 4 + j] = __uint_as_float(we[j]);
        } else {
          unpack2<T>(wa[j], vd[2 * j], vd[2 * j + 1]);
          unpack2<T>(wb[j], vg[2 * j], vg[2 * j + 1]);
          unpack2<T>(we[j], vu[2 * j], vu[2 * j + 1]);
        }
      }
    }
    if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
      for (int j = 0; j < 8; ++j) largest = fmaxf(largest, fmaxf(fabsf(vg[j]), fabsf(vu[j])));
      if (isinf(largest)) {
        const T* x = static_cast<const T*>(src.x) + row * src.ld_x;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (c + j >= cols) continue;
          if (isinf(vg[j])) vg[j] = dot_f16(x, static_cast<const T*>(src.gate) + (c + j) * src.ld_gate, src.hidden);
          if (isinf(vu[j])) vu[j] = dot_f16(x, static_cast<const T*>(src.up) + (c + j) * src.ld_up, src.hidden);
        }
      }
    }
    if (!dh_vec) {
#pragma unroll
      for (int j = 0; j < 8; ++j) vd[j] = c + j < cols ? Conv<T>::to_f(dh[row * ld_dh + c + j]) : 0.f;
    }
    float og[8], ou[8];
    with_act(act, [&](auto tag) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float a, d;
        glu_act<decltype(tag)::kAct, sizeof(T) == 4>(vg[j], a, d);
        const bool on = c + j < cols;
        og[j] = on ? vd[j] * vu[j] * d : 0.f;
        ou[j] = on ? vd[j] * a : 0.f;
      }
    });
    T* o = out + row * 2 * cols_pad + c;
#pragma unroll
    for (int k = 0; k < Q; ++k) {
      if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4*>(o)[k] = make_float4(og[4 * k], og[4 * k + 1], og[4 * k + 2], og[4 * k + 3]);
        reinterpret_cast<float4*>(o + cols_pad)[k] = make_float4(ou[4 * k], ou[4 * k + 1], ou[4 * k + 2], ou[4 * k + 3]);
      } else {
        *reinterpret_cast<uint4*>(o) =
            make_uint4(pack2<T>(og[0], og[1]), pack2<T>(og[2], og[3]), pack2<T>(og[4], og[5]), pack2<T>(og[6], og[7]));
        *reinterpret_cast<uint4*>(o + cols_pad) =
            make_uint4(pack2<T>(ou[0], ou[1]), pack2<T>(ou[2], ou[3]), pack2<T>(ou[4], ou[5]), pack2<T>(ou[6], ou[7]));
      }
    }
  }
}

// Rows of 16-bit elements copied into rows of cols_pad (a multiple of 8) that end in zeros.
struct PadRowsParams {
  const uint16_t* src[3];
  uint16_t* dst[3];
  int64_t ld[3];
  int64_t last[3];       // vectors of matrices 0 .. i
  int64_t cols, cols_pad;
  int32_t count;
};

static __global__ void __launch_bounds__(256) pad_rows_kernel(const __grid_constant__ PadRowsParams p) {
  const int64_t vecs = p.cols_pad / 8;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < p.last[p.count - 1];
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    int m = 0;
    while (i >= p.last[m]) ++m;
    const int64_t at = i - (m ? p.last[m - 1] : 0), row = at / vecs, c = (at - row * vecs) * 8;
    const uint16_t* s = p.src[m] + row * p.ld[m] + c;
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t a = c + 2 * j < p.cols ? s[2 * j] : 0u, b = c + 2 * j + 1 < p.cols ? s[2 * j + 1] : 0u;
      w[j] = a | b << 16;
    }
    reinterpret_cast<uint4*>(p.dst[m])[at] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// sum_split_kernel for results whose rows are no multiple of 8: partials [split][rows][cols_pad], out [rows, cols].
template <typename T>
__global__ void __launch_bounds__(256) sum_split_rows_kernel(const float* part, int splits, int64_t rows, int64_t cols,
                                                             int64_t cols_pad, T* out) {
  const int64_t total = rows * cols;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t row = i / cols, at = row * cols_pad + (i - row * cols);
    float v = part[at];
    for (int k = 1; k < splits; ++k) v += part[k * rows * cols_pad + at];
    out[i] = Conv<T>::from_f(v);
  }
}

}  // namespace orda
