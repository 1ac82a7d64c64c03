// Rotary positions of queries and keys in one pass, alone or after a per-head RMS norm, and the
// backward pass of the normed form.
//
// A pair (a, b) of a head at position p turns by the angle p * theta_i:
//   a' = m (a cos - b sin),  b' = m (b cos + a sin)
// and the backward pass of the plain rotation is the rotation by the negative angle. With the norm,
// n = x r, r = rsqrt(mean x^2 + eps), y = R(w n):
//   dz = R^T dy,  dw = sum over heads and tokens of dz n,  e = w dz,  dx = r (e - n mean(e n)).
//
// Angles: theta_i / 2 pi is held in 64 bits, p times it is reduced to [-1/2, 1/2] turns in 64 bits
// and only then rounded to 32, so the angle is off by less than 2e-7 rad at any position below 2^31
// (a 32-bit product is already off by 0.06 rad at position 1e6). No table: a warp computes a token's
// angles once for the heads that it turns.
//
// What bounds it: memory. Each head's values are read and written once, 16-byte vectors, and a lane's
// cosines, sines and norm weights stay in registers over the heads of the token.
#pragma once

#include "distill_common.cuh"
#include "orda_b200_student.h"

namespace orda {

constexpr int kRotWarps = 4;                              // warps per block
constexpr int kRotMaxPairs = ORDA_ROTARY_MAX_DIM / 2;

struct RotaryParams {
  const void* x[2];
  const void* dy[2];
  void* out[2];
  const void* w[2];
  int64_t xs[2][3], os[2][3], ds[2][3];
  const void* pos;
  int64_t ps[2];
  float* dw_partial;              // [grid][2][D]
  int32_t seq, tokens;
  int32_t heads[2];
  int32_t units[2];               // work units of a token: groups of heads_per_unit query / key heads
  int32_t heads_per_unit;
  int32_t head_dim, rotary_dim;
  int32_t lanes;                  // lanes per head: a power of two <= 32
  int32_t pos64, interleaved, w_dtype;
  float magnitude, sin_sign, eps;
  double turns[kRotMaxPairs];     // theta_i / (2 pi)
};

__device__ __forceinline__ float load_weight(const void* w, int dtype, int i) {
  if (dtype == ORDA_F32) return static_cast<const float*>(w)[i];
  if (dtype == ORDA_F16) return __half2float(static_cast<const __half*>(w)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
}

// V consecutive elements as floats; the address is a multiple of V * sizeof(T) bytes (at most 16)
template <typename T, int V>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[V]) {
  if constexpr (V * sizeof(T) >= 16) {
#pragma unroll
    for (int q = 0; q < static_cast<int>(V * sizeof(T) / 16); ++q) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(p) + q);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[q * 4 + i] = __uint_as_float(w[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) unpack2<T>(w[i], v[q * 8 + 2 * i], v[q * 8 + 2 * i + 1]);
      }
    }
  } else if constexpr (V == 2 && sizeof(T) == 2) {
    unpack2<T>(__ldg(reinterpret_cast<const uint32_t*>(p)), v[0], v[1]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = Conv<T>::to_f(p[i]);
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[V]) {
  if constexpr (V * sizeof(T) >= 16) {
#pragma unroll
    for (int q = 0; q < static_cast<int>(V * sizeof(T) / 16); ++q) {
      uint4 u;
      if constexpr (sizeof(T) == 4) {
        u = make_uint4(__float_as_uint(v[q * 4]), __float_as_uint(v[q * 4 + 1]), __float_as_uint(v[q * 4 + 2]),
                       __float_as_uint(v[q * 4 + 3]));
      } else {
        u = make_uint4(pack2<T>(v[q * 8], v[q * 8 + 1]), pack2<T>(v[q * 8 + 2], v[q * 8 + 3]),
                       pack2<T>(v[q * 8 + 4], v[q * 8 + 5]), pack2<T>(v[q * 8 + 6], v[q * 8 + 7]));
      }
      reinterpret_cast<uint4*>(p)[q] = u;
    }
  } else if constexpr (V == 2 && sizeof(T) == 2) {
    *reinterpret_cast<uint32_t*>(p) = pack2<T>(v[0], v[1]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] = Conv<T>::from_f(v[i]);
  }
}

// Where a lane's slot (2 V elements of a head) lies: a rotated slot holds V whole pairs (half layout:
// the first vector's elements with the second's; interleaved: neighbours), the slots behind rotary_dim
// hold 2 V values that pass through.
template <int V>
struct Slot {
  int a, b;       // first element of the two V-vectors
  bool on, on_b;  // inside the head (V = 1 and an odd head size: the last slot has no b)
  bool turned;
};

template <int V>
__device__ __forceinline__ Slot<V> slot_of(const RotaryParams& p, int s) {
  Slot<V> r;
  const int rotated = p.rotary_dim / (2 * V);
  r.turned = s < rotated;
  if (r.turned) {
    r.a = p.interleaved ? s * 2 * V : s * V;
    r.b = p.interleaved ? s * 2 * V + V : p.rotary_dim / 2 + s * V;
  } else {
    r.a = p.rotary_dim + (s - rotated) * 2 * V;
    r.b = r.a + V;
  }
  r.on = r.a < p.head_dim;
  r.on_b = r.b < p.head_dim;
  return r;
}

// The angles of one token, by its warp: cs[i] = magnitude * (cos, +-sin) of pair i.
__device__ __forceinline__ void token_angles(const RotaryParams& p, int b, int t, int lane, float2* cs) {
  const int64_t at = b * p.ps[0] + t * p.ps[1];
  const double pos = p.pos64 ? static_cast<double>(static_cast<const int64_t*>(p.pos)[at])
                             : static_cast<double>(static_cast<const int32_t*>(p.pos)[at]);
  for (int i = lane; i < p.rotary_dim / 2; i += 32) {
    double turn = pos * p.turns[i];
    turn -= rint(turn);
    float s, c;
    sincospif(2.f * static_cast<float>(turn), &s, &c);
    cs[i] = make_float2(p.magnitude * c, p.magnitude * p.sin_sign * s);
  }
  __syncwarp();
}

// One slot turned in place by the (cos, sin) of its V pairs.
template <int V>
__device__ __forceinline__ void turn_slot(float (&a)[V], float (&b)[V], const float2 (&cs)[V], bool interleaved) {
  if (V == 1 || !interleaved) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float ya = a[i] * cs[i].x - b[i] * cs[i].y;
      b[i] = b[i] * cs[i].x + a[i] * cs[i].y;
      a[i] = ya;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float2 c1 = cs[i], c2 = cs[V / 2 + i];
      const float ya = a[2 * i] * c1.x - a[2 * i + 1] * c1.y;
      a[2 * i + 1] = a[2 * i + 1] * c1.x + a[2 * i] * c1.y;
      a[2 * i] = ya;
      const float yb = b[2 * i] * c2.x - b[2 * i + 1] * c2.y;
      b[2 * i + 1] = b[2 * i + 1] * c2.x + b[2 * i] * c2.y;
      b[2 * i] = yb;
    }
  }
}

__device__ __forceinline__ float group_sum(float v, int lanes) {
  for (int o = lanes / 2; o > 0; o /= 2) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// slots a lane may have to hold (1 with 8-element vectors: 32 lanes cover 512 elements)
template <int V>
constexpr int rotary_slots_per_lane() {
  return kRotMaxPairs / (32 * V);
}

template <typename T, int V, bool NORM>
__global__ void __launch_bounds__(32 * kRotWarps) rotary_forward_kernel(const __grid_constant__ RotaryParams p) {
  constexpr int NS = rotary_slots_per_lane<V>();
  __shared__ float2 cs_all[kRotWarps][kRotMaxPairs];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  float2* cs_token = cs_all[warp];
  const int per_token = p.units[0] + p.units[1];
  const int64_t total = static_cast<int64_t>(p.tokens) * per_token;
  const int sub = lane / p.lanes, sl = lane % p.lanes, at_once = 32 / p.lanes;
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * kRotWarps + warp; u < total;
       u += static_cast<int64_t>(gridDim.x) * kRotWarps) {
    const int token = static_cast<int>(u / per_token);
    int g = static_cast<int>(u - static_cast<int64_t>(token) * per_token);
    const int which = g >= p.units[0];
    if (which) g -= p.units[0];
    const int b = token / p.seq, t = token - b * p.seq;
    __syncwarp();  // the previous unit's angles have been read
    token_angles(p, b, t, lane, cs_token);
    Slot<V> slot[NS];
    float2 cs[NS][V];
    float wa[NS][V], wb[NS][V];
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      const int s = sl + n * p.lanes;
      slot[n] = slot_of<V>(p, s);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        cs[n][i] = slot[n].turned ? cs_token[s * V + i] : make_float2(1.f, 0.f);
        if constexpr (NORM) {
          wa[n][i] = slot[n].on ? load_weight(p.w[which], p.w_dtype, slot[n].a + i) : 0.f;
          wb[n][i] = slot[n].on_b ? load_weight(p.w[which], p.w_dtype, slot[n].b + i) : 0.f;
        }
      }
    }
    const T* x = static_cast<const T*>(p.x[which]) + b * p.xs[which][0] + t * p.xs[which][1];
    T* out = static_cast<T*>(p.out[which]) + b * p.os[which][0] + t * p.os[which][1];
    const int h_end = min(p.heads[which], (g + 1) * p.heads_per_unit);
    for (int h0 = g * p.heads_per_unit; h0 < h_end; h0 += at_once) {
      const int h = h0 + sub;
      const bool live = h < h_end;
      const T* xh = x + h * p.xs[which][2];
      T* oh = out + h * p.os[which][2];
      float va[NS][V], vb[NS][V];
      float ss = 0.f;
#pragma unroll
      for (int n = 0; n < NS; ++n) {
#pragma unroll
        for (int i = 0; i < V; ++i) va[n][i] = vb[n][i] = 0.f;
        if (live && slot[n].on) load_vec<T, V>(xh + slot[n].a, va[n]);
        if (live && slot[n].on_b) load_vec<T, V>(xh + slot[n].b, vb[n]);
        if constexpr (NORM) {
#pragma unroll
          for (int i = 0; i < V; ++i) ss += va[n][i] * va[n][i] + vb[n][i] * vb[n][i];
        }
      }
      float r = 1.f;
      if constexpr (NORM) r = rsqrtf(group_sum(ss, p.lanes) / p.head_dim + p.eps);
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        if constexpr (NORM) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            va[n][i] *= r * wa[n][i];
            vb[n][i] *= r * wb[n][i];
          }
        }
        turn_slot<V>(va[n], vb[n], cs[n], p.interleaved != 0);
        if (live && slot[n].on) store_vec<T, V>(oh + slot[n].a, va[n]);
        if (live && slot[n].on_b) store_vec<T, V>(oh + slot[n].b, vb[n]);
      }
    }
  }
}

// Backward of the normed form. Each lane adds up the weight gradients of its elements over every head
// it meets, the block adds its warps' and head groups' sums in a fixed order and writes one partial row;
// norm_weight_grad_kernel adds the blocks' rows, again in a fixed order: the same inputs give the same
// bits.
template <typename T, int V>
__global__ void __launch_bounds__(32 * kRotWarps) qk_norm_rotary_backward_kernel(const __grid_constant__ RotaryParams p) {
  constexpr int NS = rotary_slots_per_lane<V>();
  __shared__ float2 cs_all[kRotWarps][kRotMaxPairs];
  __shared__ float dw_s[kRotWarps][ORDA_ROTARY_MAX_DIM];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  float2* cs_token = cs_all[warp];
  const int sub = lane / p.lanes, sl = lane % p.lanes, at_once = 32 / p.lanes;
  for (int which = 0; which < 2; ++which) {
    const int64_t total = static_cast<int64_t>(p.tokens) * p.units[which];
    Slot<V> slot[NS];
    float wa[NS][V], wb[NS][V], dwa[NS][V], dwb[NS][V];
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      slot[n] = slot_of<V>(p, sl + n * p.lanes);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        wa[n][i] = slot[n].on ? load_weight(p.w[which], p.w_dtype, slot[n].a + i) : 0.f;
        wb[n][i] = slot[n].on_b ? load_weight(p.w[which], p.w_dtype, slot[n].b + i) : 0.f;
        dwa[n][i] = dwb[n][i] = 0.f;
      }
    }
    for (int64_t u = static_cast<int64_t>(blockIdx.x) * kRotWarps + warp; u < total;
         u += static_cast<int64_t>(gridDim.x) * kRotWarps) {
      const int token = static_cast<int>(u / p.units[which]);
      const int g = static_cast<int>(u - static_cast<int64_t>(token) * p.units[which]);
      const int b = token / p.seq, t = token - b * p.seq;
      __syncwarp();
      token_angles(p, b, t, lane, cs_token);
      float2 cs[NS][V];
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int i = 0; i < V; ++i)
          cs[n][i] = slot[n].turned ? cs_token[(sl + n * p.lanes) * V + i] : make_float2(1.f, 0.f);
      const T* x = static_cast<const T*>(p.x[which]) + b * p.xs[which][0] + t * p.xs[which][1];
      const T* dy = static_cast<const T*>(p.dy[which]) + b * p.ds[which][0] + t * p.ds[which][1];
      T* out = static_cast<T*>(p.out[which]) + b * p.os[which][0] + t * p.os[which][1];
      const int h_end = min(p.heads[which], (g + 1) * p.heads_per_unit);
      for (int h0 = g * p.heads_per_unit; h0 < h_end; h0 += at_once) {
        const int h = h0 + sub;
        const bool live = h < h_end;
        const T* xh = x + h * p.xs[which][2];
        const T* dh = dy + h * p.ds[which][2];
        T* oh = out + h * p.os[which][2];
        float xa[NS][V], xb[NS][V], za[NS][V], zb[NS][V];
        float ss = 0.f, ex = 0.f;  // sum x^2, sum (w dz) x
#pragma unroll
        for (int n = 0; n < NS; ++n) {
#pragma unroll
          for (int i = 0; i < V; ++i) xa[n][i] = xb[n][i] = za[n][i] = zb[n][i] = 0.f;
          if (live && slot[n].on) {
            load_vec<T, V>(xh + slot[n].a, xa[n]);
            load_vec<T, V>(dh + slot[n].a, za[n]);
          }
          if (live && slot[n].on_b) {
            load_vec<T, V>(xh + slot[n].b, xb[n]);
            load_vec<T, V>(dh + slot[n].b, zb[n]);
          }
          turn_slot<V>(za[n], zb[n], cs[n], p.interleaved != 0);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            ss += xa[n][i] * xa[n][i] + xb[n][i] * xb[n][i];
            ex += za[n][i] * wa[n][i] * xa[n][i] + zb[n][i] * wb[n][i] * xb[n][i];
          }
        }
        ss = group_sum(ss, p.lanes);
        ex = group_sum(ex, p.lanes);
        const float r = rsqrtf(ss / p.head_dim + p.eps);
        const float m = r * r * ex / p.head_dim;  // r mean(e n)
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          float ga[V], gb[V];
#pragma unroll
          for (int i = 0; i < V; ++i) {
            dwa[n][i] += za[n][i] * (xa[n][i] * r);
            dwb[n][i] += zb[n][i] * (xb[n][i] * r);
            ga[i] = r * (za[n][i] * wa[n][i] - xa[n][i] * m);
            gb[i] = r * (zb[n][i] * wb[n][i] - xb[n][i] * m);
          }
          if (live && slot[n].on) store_vec<T, V>(oh + slot[n].a, ga);
          if (live && slot[n].on_b) store_vec<T, V>(oh + slot[n].b, gb);
        }
      }
    }
    // head groups of the warp, then the warps of the block
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float a = dwa[n][i], b = dwb[n][i];
        for (int o = p.lanes; o < 32; o *= 2) {
          a += __shfl_xor_sync(0xffffffffu, a, o);
          b += __shfl_xor_sync(0xffffffffu, b, o);
        }
        if (sub == 0 && slot[n].on) dw_s[warp][slot[n].a + i] = a;
        if (sub == 0 && slot[n].on_b) dw_s[warp][slot[n].b + i] = b;
      }
    __syncthreads();
    float* row = p.dw_partial + (static_cast<int64_t>(blockIdx.x) * 2 + which) * p.head_dim;
    for (int i = threadIdx.x; i < p.head_dim; i += blockDim.x) {
      float v = 0.f;
#pragma unroll
      for (int k = 0; k < kRotWarps; ++k) v += dw_s[k][i];
      row[i] = v;
    }
  }
}

// dweight[which][i] = sum over the blocks' partial rows; one block per 32 columns of one weight.
static __global__ void __launch_bounds__(256) norm_weight_grad_kernel(const float* partial, int rows, int head_dim,
                                                                      int dtype, void* dwq, void* dwk) {
  __shared__ float acc[8][32];
  const int which = blockIdx.y, col = blockIdx.x * 32 + threadIdx.x % 32, part = threadIdx.x / 32;
  float v = 0.f;
  if (col < head_dim)
    for (int r = part; r < rows; r += 8) v += partial[(static_cast<int64_t>(r) * 2 + which) * head_dim + col];
  acc[part][threadIdx.x % 32] = v;
  __syncthreads();
  if (part != 0 || col >= head_dim) return;
  for (int k = 1; k < 8; ++k) v += acc[k][threadIdx.x];
  void* out = which ? dwk : dwq;
  if (dtype == ORDA_F32) static_cast<float*>(out)[col] = v;
  else if (dtype == ORDA_F16) static_cast<__half*>(out)[col] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(out)[col] = __float2bfloat16_rn(v);
}

}  // namespace orda
