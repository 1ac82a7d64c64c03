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
  int32_t units[2];               // work units of a token: groups of heads_per_unit heads. Forward: [0] over query
                                  // and key heads together; backward: over the query heads, over the key heads
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

// V consecutive elements as they lie in memory; the address is a multiple of V * sizeof(T) bytes (at
// most 16). Kept packed so that a lane can have several heads in flight.
template <typename T, int V>
struct Raw {
  static constexpr int kBytes = V * static_cast<int>(sizeof(T));
  static constexpr int kWords = kBytes >= 4 ? kBytes / 4 : 1;
  uint32_t w[kWords];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0u;
  }
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kBytes >= 16) {
#pragma unroll
      for (int q = 0; q < kBytes / 16; ++q) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(p) + q);
        w[4 * q] = u.x; w[4 * q + 1] = u.y; w[4 * q + 2] = u.z; w[4 * q + 3] = u.w;
      }
    } else if constexpr (kBytes == 8) {
      const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
      w[0] = u.x; w[1] = u.y;
    } else if constexpr (kBytes == 4) {
      w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
    } else {
      w[0] = __ldg(reinterpret_cast<const unsigned short*>(p));
    }
  }
  __device__ __forceinline__ void unpack(float (&v)[V]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = __uint_as_float(w[i]);
    } else if constexpr (V == 1) {
      float high;
      unpack2<T>(w[0], v[0], high);
    } else {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) unpack2<T>(w[i], v[2 * i], v[2 * i + 1]);
    }
  }
};

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
  } else if constexpr (V == 2) {
    *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
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

// Where a warp keeps the (cos, sin) of a token's pairs, and a block its norm weights, in shared memory:
// the V of a slot as 16-byte pieces, piece k of every slot side by side, so that the lanes' 16-byte reads
// of one piece are consecutive (64 bytes apart they would meet in the same banks four by four).
template <int V>
__device__ __forceinline__ int pair_at(int slots, int pair) {
  if constexpr (V < 4) {
    return pair;
  } else {
    const int s = pair / V, i = pair % V;
    return ((i / 2) * slots + s) * 2 + i % 2;
  }
}

__device__ __forceinline__ int64_t token_position(const RotaryParams& p, int b, int t) {
  const int64_t at = b * p.ps[0] + t * p.ps[1];
  return p.pos64 ? __ldg(static_cast<const long long*>(p.pos) + at) : __ldg(static_cast<const int32_t*>(p.pos) + at);
}

// The angles of one token, by its warp: magnitude * (cos, +-sin) of each pair.
template <int V>
__device__ __forceinline__ void token_angles(const RotaryParams& p, int64_t position, int lane, float2* cs) {
  const double pos = static_cast<double>(position);
  const int rotated = p.rotary_dim / (2 * V);
  for (int i = lane; i < p.rotary_dim / 2; i += 32) {
    double turn = pos * p.turns[i];
    turn -= rint(turn);
    float s, c;
    sincospif(2.f * static_cast<float>(turn), &s, &c);
    cs[pair_at<V>(rotated, i)] = make_float2(p.magnitude * c, p.magnitude * p.sin_sign * s);
  }
  __syncwarp();
}

// The (cos, sin) of slot s, (1, 0) where the slot passes through.
template <int V>
__device__ __forceinline__ void slot_angles(const RotaryParams& p, const float2* cs, int s, bool turned,
                                            float2 (&out)[V]) {
  const int rotated = p.rotary_dim / (2 * V);
  if constexpr (V < 4) {
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = turned ? cs[s * V + i] : make_float2(1.f, 0.f);
  } else {
#pragma unroll
    for (int k = 0; k < V / 2; ++k) {
      const float4 u = turned ? reinterpret_cast<const float4*>(cs)[k * rotated + s] : make_float4(1.f, 0.f, 1.f, 0.f);
      out[2 * k] = make_float2(u.x, u.y);
      out[2 * k + 1] = make_float2(u.z, u.w);
    }
  }
}

// (weight of a, weight of b) of slot s
template <int V>
__device__ __forceinline__ void slot_weights(const float2* w_s, int slots, int s, float2 (&out)[V]) {
  if constexpr (V < 4) {
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = w_s[s * V + i];
  } else {
#pragma unroll
    for (int k = 0; k < V / 2; ++k) {
      const float4 u = reinterpret_cast<const float4*>(w_s)[k * slots + s];
      out[2 * k] = make_float2(u.x, u.y);
      out[2 * k + 1] = make_float2(u.z, u.w);
    }
  }
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

// Where a warp stands: a unit (a token's group of heads) and the pass over its heads, at_once heads a pass.
// Both kernels load the values of the next pass, of the next unit if need be, before they work on the
// current one: a warp always has a pass in flight, and a token's angles are formed while its first
// values arrive.
struct RotaryStep {
  int64_t unit;
  int head;         // first head of the pass
  int end;          // behind the unit's last head
  int64_t xq, xk;   // element offset of the token in the two inputs
  int64_t position;
  int b, t;
};

template <typename T, int V, bool NORM>
__global__ void __launch_bounds__(32 * kRotWarps) rotary_forward_kernel(const __grid_constant__ RotaryParams p) {
  constexpr int NS = rotary_slots_per_lane<V>();
  __shared__ __align__(16) float2 cs_all[kRotWarps][kRotMaxPairs];
  __shared__ __align__(16) float2 w_s[NORM ? 2 : 1][NORM ? kRotMaxPairs : 1];  // (of a, of b) of each slot
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  float2* cs_token = cs_all[warp];
  const int heads = p.heads[0] + p.heads[1];
  const int64_t total = static_cast<int64_t>(p.tokens) * p.units[0];
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kRotWarps;
  const int sub = lane / p.lanes, sl = lane % p.lanes, at_once = 32 / p.lanes;
  const int slots = NS * p.lanes;
  Slot<V> slot[NS];
#pragma unroll
  for (int n = 0; n < NS; ++n) slot[n] = slot_of<V>(p, sl + n * p.lanes);
  if constexpr (NORM) {
    for (int i = threadIdx.x; i < slots * V; i += blockDim.x) {
      const Slot<V> q = slot_of<V>(p, i / V);
      const int e = i % V;
#pragma unroll
      for (int w = 0; w < 2; ++w)
        w_s[w][pair_at<V>(slots, i)] = make_float2(q.on ? load_weight(p.w[w], p.w_dtype, q.a + e) : 0.f,
                                                   q.on_b ? load_weight(p.w[w], p.w_dtype, q.b + e) : 0.f);
    }
    __syncthreads();
  }
  auto begin = [&](int64_t unit) {
    RotaryStep st;
    st.unit = unit;
    const int token = static_cast<int>(unit / p.units[0]);
    const int g = static_cast<int>(unit - static_cast<int64_t>(token) * p.units[0]);
    st.b = token / p.seq;
    st.t = token - st.b * p.seq;
    st.head = g * p.heads_per_unit;
    st.end = min(heads, st.head + p.heads_per_unit);
    st.xq = st.b * p.xs[0][0] + st.t * p.xs[0][1];
    st.xk = st.b * p.xs[1][0] + st.t * p.xs[1][1];
    st.position = token_position(p, st.b, st.t);
    return st;
  };
  Raw<T, V> ra[NS], rb[NS];
  auto fetch = [&](const RotaryStep& st) {
    const int h = st.head + sub;
    const bool key = h >= p.heads[0];
    const T* x = key ? static_cast<const T*>(p.x[1]) + st.xk + (h - p.heads[0]) * p.xs[1][2]
                     : static_cast<const T*>(p.x[0]) + st.xq + h * p.xs[0][2];
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      ra[n].clear();
      rb[n].clear();
      if (h < st.end && slot[n].on) ra[n].load(x + slot[n].a);
      if (h < st.end && slot[n].on_b) rb[n].load(x + slot[n].b);
    }
  };
  int64_t unit = static_cast<int64_t>(blockIdx.x) * kRotWarps + warp;
  if (unit >= total) return;
  RotaryStep next = begin(unit);
  fetch(next);
  float2 cs[NS][V];
  bool fresh = true;  // the pass is its unit's first
  while (true) {
    const RotaryStep st = next;
    Raw<T, V> ca[NS], cb[NS];
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      ca[n] = ra[n];
      cb[n] = rb[n];
    }
    const bool same = st.head + at_once < st.end;
    const bool more = same || st.unit + stride < total;
    if (same) next.head += at_once;
    else if (more) next = begin(st.unit + stride);
    if (more) fetch(next);
    if (fresh) {
      __syncwarp();  // the previous unit's angles have been read
      token_angles<V>(p, st.position, lane, cs_token);
#pragma unroll
      for (int n = 0; n < NS; ++n) slot_angles<V>(p, cs_token, sl + n * p.lanes, slot[n].turned, cs[n]);
    }
    const int h = st.head + sub;
    const bool live = h < st.end, key = h >= p.heads[0];
    T* out = key ? static_cast<T*>(p.out[1]) + st.b * p.os[1][0] + st.t * p.os[1][1] + (h - p.heads[0]) * p.os[1][2]
                 : static_cast<T*>(p.out[0]) + st.b * p.os[0][0] + st.t * p.os[0][1] + h * p.os[0][2];
    float va[NS][V], vb[NS][V];
    float ss = 0.f;
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      ca[n].unpack(va[n]);
      cb[n].unpack(vb[n]);
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
        float2 w[V];
        slot_weights<V>(w_s[key], slots, sl + n * p.lanes, w);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          va[n][i] *= r * w[i].x;
          vb[n][i] *= r * w[i].y;
        }
      }
      turn_slot<V>(va[n], vb[n], cs[n], p.interleaved != 0);
      if (live && slot[n].on) store_vec<T, V>(out + slot[n].a, va[n]);
      if (live && slot[n].on_b) store_vec<T, V>(out + slot[n].b, vb[n]);
    }
    if (!more) break;
    fresh = !same;
  }
}

// Backward of the normed form. Each lane adds up the weight gradients of its elements over every head
// it meets, the block adds its warps' and head groups' sums in a fixed order and writes one partial row;
// norm_weight_grad_kernel adds the blocks' rows, again in a fixed order: the same inputs give the same
// bits. Cosines, sines and weights stay in shared memory: in registers they would leave room for half
// as many warps.
template <typename T, int V>
__global__ void __launch_bounds__(32 * kRotWarps, 4)
    qk_norm_rotary_backward_kernel(const __grid_constant__ RotaryParams p) {
  constexpr int NS = rotary_slots_per_lane<V>();
  __shared__ __align__(16) float2 cs_all[kRotWarps][kRotMaxPairs];
  __shared__ __align__(16) float2 w_s[kRotMaxPairs];  // (weight of a, weight of b) of each slot
  __shared__ float dw_s[kRotWarps][ORDA_ROTARY_MAX_DIM];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  float2* cs_token = cs_all[warp];
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kRotWarps;
  const int sub = lane / p.lanes, sl = lane % p.lanes, at_once = 32 / p.lanes;
  const int slots = NS * p.lanes;
  Slot<V> slot[NS];
#pragma unroll
  for (int n = 0; n < NS; ++n) slot[n] = slot_of<V>(p, sl + n * p.lanes);
  for (int which = 0; which < 2; ++which) {
    __syncthreads();  // the previous weights and sums have been read
    for (int i = threadIdx.x; i < slots * V; i += blockDim.x) {
      const Slot<V> q = slot_of<V>(p, i / V);
      const int e = i % V;
      w_s[pair_at<V>(slots, i)] = make_float2(q.on ? load_weight(p.w[which], p.w_dtype, q.a + e) : 0.f,
                                              q.on_b ? load_weight(p.w[which], p.w_dtype, q.b + e) : 0.f);
    }
    __syncthreads();
    const int64_t total = static_cast<int64_t>(p.tokens) * p.units[which];
    float dwa[NS][V], dwb[NS][V];
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int i = 0; i < V; ++i) dwa[n][i] = dwb[n][i] = 0.f;
    auto begin = [&](int64_t unit) {
      RotaryStep st;
      st.unit = unit;
      const int token = static_cast<int>(unit / p.units[which]);
      const int g = static_cast<int>(unit - static_cast<int64_t>(token) * p.units[which]);
      st.b = token / p.seq;
      st.t = token - st.b * p.seq;
      st.head = g * p.heads_per_unit;
      st.end = min(p.heads[which], st.head + p.heads_per_unit);
      st.xq = st.b * p.xs[which][0] + st.t * p.xs[which][1];
      st.xk = st.b * p.ds[which][0] + st.t * p.ds[which][1];  // (of dy)
      st.position = token_position(p, st.b, st.t);
      return st;
    };
    Raw<T, V> rx[NS][2], rz[NS][2];
    auto fetch = [&](const RotaryStep& st) {
      const int h = st.head + sub;
      const T* x = static_cast<const T*>(p.x[which]) + st.xq + h * p.xs[which][2];
      const T* z = static_cast<const T*>(p.dy[which]) + st.xk + h * p.ds[which][2];
#pragma unroll
      for (int n = 0; n < NS; ++n) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          rx[n][j].clear();
          rz[n][j].clear();
        }
        if (h < st.end && slot[n].on) {
          rx[n][0].load(x + slot[n].a);
          rz[n][0].load(z + slot[n].a);
        }
        if (h < st.end && slot[n].on_b) {
          rx[n][1].load(x + slot[n].b);
          rz[n][1].load(z + slot[n].b);
        }
      }
    };
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * kRotWarps + warp;
    RotaryStep next{};
    bool more = unit < total, fresh = true;
    if (more) {
      next = begin(unit);
      fetch(next);
    }
    while (more) {
      const RotaryStep st = next;
      Raw<T, V> cx[NS][2], cz[NS][2];
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          cx[n][j] = rx[n][j];
          cz[n][j] = rz[n][j];
        }
      const bool same = st.head + at_once < st.end;
      more = same || st.unit + stride < total;
      if (same) next.head += at_once;
      else if (more) next = begin(st.unit + stride);
      if (more) fetch(next);
      if (fresh) {
        __syncwarp();  // the previous unit's angles have been read
        token_angles<V>(p, st.position, lane, cs_token);
      }
      fresh = !same;
      const int h = st.head + sub;
      const bool live = h < st.end;
      T* out = static_cast<T*>(p.out[which]) + st.b * p.os[which][0] + st.t * p.os[which][1] + h * p.os[which][2];
      float xa[NS][V], xb[NS][V], za[NS][V], zb[NS][V];
      float ss = 0.f, ex = 0.f;  // sum x^2, sum (w dz) x
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        const int s = sl + n * p.lanes;
        cx[n][0].unpack(xa[n]);
        cx[n][1].unpack(xb[n]);
        cz[n][0].unpack(za[n]);
        cz[n][1].unpack(zb[n]);
        float2 cs[V], w[V];
        slot_angles<V>(p, cs_token, s, slot[n].turned, cs);
        slot_weights<V>(w_s, slots, s, w);
        turn_slot<V>(za[n], zb[n], cs, p.interleaved != 0);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          ss += xa[n][i] * xa[n][i] + xb[n][i] * xb[n][i];
          ex += za[n][i] * w[i].x * xa[n][i] + zb[n][i] * w[i].y * xb[n][i];
        }
      }
      ss = group_sum(ss, p.lanes);
      ex = group_sum(ex, p.lanes);
      const float r = rsqrtf(ss / p.head_dim + p.eps);
      const float m = r * r * ex / p.head_dim;  // r mean(e n)
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        float2 w[V];
        slot_weights<V>(w_s, slots, sl + n * p.lanes, w);
        float ga[V], gb[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          dwa[n][i] += za[n][i] * (xa[n][i] * r);
          dwb[n][i] += zb[n][i] * (xb[n][i] * r);
          ga[i] = r * (za[n][i] * w[i].x - xa[n][i] * m);
          gb[i] = r * (zb[n][i] * w[i].y - xb[n][i] * m);
        }
        if (live && slot[n].on) store_vec<T, V>(out + slot[n].a, ga);
        if (live && slot[n].on_b) store_vec<T, V>(out + slot[n].b, gb);
      }
    }
    // head groups of the warp, then the warps of the block
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
