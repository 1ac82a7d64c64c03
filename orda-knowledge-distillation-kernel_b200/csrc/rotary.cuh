// Rotary positions of queries and keys in one pass, alone or after a per-head RMS norm, and the
// backward pass of the normed form.
//
// A pair (a, b) of a head at position p turns by the angle p * theta_i:
//   a' = m (a cos - b sin),  b' = m (b cos + a sin)
// and the backward pass of the plain rotation is the rotation by the negative angle. With the norm,
// n = x r, r = rsqrt(mean x^2 + eps), y = R(w n):
//   dz = R^T dy,  dw = sum over heads and tokens of dz n,  e = w dz,  dx = r (e - n mean(e n)).
//
// Angles: theta_i / 2 pi is held as a 64-bit fraction of a turn, and the low 64 bits of its product with
// the position are the angle modulo one turn, off by |p| 2^-65 turns plus the rounding of theta_i. The
// top 32 of them go to fp32, so the angle is off by less than 1e-7 rad at any position below 2^31 (a
// 32-bit float product is already off by 0.06 rad at position 1e6); for fp32 tensors, where a sine near zero
// would show it, cosine and sine are corrected by the rest. No table and no fp64 arithmetic: a warp computes a
// token's angles once for the heads that it turns.
//
// What bounds it: memory, and close behind it the issue of instructions (61-67% of the slots). Each head's
// values are read and written once in 16-byte vectors, a token's angles are formed once. In bf16: 32768 tokens
// of 10 heads of 128 are rotated in 33.0 us (5.1 TB/s), 16384 of 40 normed and rotated in 60 us (5.6 TB/s), and
// back in 96 us (5.2 TB/s) and 5 for the weights' sums.
#pragma once

#include <type_traits>

#include "distill_common.cuh"
#include "orda_b200_student.h"

namespace orda {

constexpr int kRotWarps = 4;                              // warps per block
constexpr int kRotMaxPairs = ORDA_ROTARY_MAX_DIM / 2;

// n / d for 0 <= n < 2^31 by a multiplication (Granlund and Montgomery's round-up method).
struct FastDiv {
  uint32_t d, mul, shift;
};

inline FastDiv make_fast_div(uint32_t d) {
  FastDiv f{d, 0, 0};
  while ((uint64_t(1) << f.shift) < d) ++f.shift;
  f.mul = static_cast<uint32_t>(((uint64_t(1) << 32) * ((uint64_t(1) << f.shift) - d)) / d + 1);
  return f;
}

__device__ __forceinline__ uint32_t fast_div(uint32_t n, const FastDiv& f) {
  return static_cast<uint32_t>((static_cast<uint64_t>(__umulhi(n, f.mul)) + n) >> f.shift);
}

struct RotaryParams {
  const void* x[2];
  const void* dy[2];
  void* out[2];
  const void* w[2];
  int64_t xs[2][2], os[2][2], ds[2][2];  // element strides of batch and seq
  int32_t xh[2], oh[2], dh[2];           // and of heads
  const void* pos;
  int64_t ps[2];
  float* dw_partial;              // [grid][2][D]
  int32_t tokens;
  FastDiv seq;
  int32_t heads[2];
  // Work units of a token: groups of heads_per_unit heads. Forward: [0] over query and key heads
  // together; backward: over the query heads, over the key heads.
  FastDiv units[2];
  int32_t heads_per_unit;
  int32_t head_dim, rotary_dim;
  int32_t lanes;                  // lanes per head: a power of two <= 32
  int32_t pos64, w_dtype;
  float magnitude, sin_sign, eps, inv_head_dim;
  uint64_t turns[kRotMaxPairs];   // theta_i / (2 pi) modulo 1, times 2^64
};

__device__ __forceinline__ float load_weight(const void* w, int dtype, int i) {
  if (dtype == ORDA_F32) return static_cast<const float*>(w)[i];
  if (dtype == ORDA_F16) return __half2float(static_cast<const __half*>(w)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
}

// V consecutive elements as they lie in memory; their address is a multiple of V * sizeof(T) bytes (at
// most 16).
template <typename T, int V>
struct Raw {
  static constexpr int kBytes = V * static_cast<int>(sizeof(T));
  static constexpr int kWords = kBytes >= 4 ? kBytes / 4 : 1;
  uint32_t w[kWords];

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

// Two floats of a register pair, for Blackwell's packed fp32 instructions: the kernels below would
// otherwise be bound by instruction issue (300 a pass of four 128-element heads, at 70% of the issue
// slots and half the memory rate).
typedef unsigned long long F2;
__device__ __forceinline__ F2 pk(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpk(F2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ F2 fma_v(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ F2 mul_v(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float fma_v(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ float mul_v(float a, float b) { return a * b; }

// V floats as the packed (V = 1: single) registers that these work on
template <int V>
struct Vec {
  static constexpr int N = V > 1 ? V / 2 : 1;
  using E = std::conditional_t<(V > 1), F2, float>;
  E e[N];

  static __device__ __forceinline__ E all(float x) {
    if constexpr (V > 1) return pk(x, x);
    else return x;
  }
  __device__ __forceinline__ void fill(float x) {
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = all(x);
  }
  __device__ __forceinline__ float sum() const {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (V > 1) {
        float a, b;
        unpk(e[i], a, b);
        t += a + b;
      } else {
        t += e[i];
      }
    }
    return t;
  }
  __device__ __forceinline__ void get(float (&v)[V]) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (V > 1) unpk(e[i], v[2 * i], v[2 * i + 1]);
      else v[0] = e[0];
    }
  }
  __device__ __forceinline__ void set(const float (&v)[V]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (V > 1) e[i] = pk(v[2 * i], v[2 * i + 1]);
      else e[0] = v[0];
    }
  }
};

// Where a lane's slot (2 V elements of a head) lies: two vectors of V elements at a and b. A rotated
// slot holds V whole pairs (u_i, v_i): in the half layout u is the first vector and v the second, in the
// interleaved one u are the even and v the odd elements of both. The slots behind rotary_dim hold 2 V
// values that pass through. In every case the lanes' first vectors lie side by side, and so do their
// second ones: with a lane's two vectors side by side instead, each access used half of its 32-byte
// sectors.
template <int V>
struct Slot {
  int a, b;
  bool on, on_b;  // inside the head (V = 1 and an odd head size: the last slot has no b)
  bool turned;
};

template <int V, bool IL>
__device__ __forceinline__ Slot<V> slot_of(const RotaryParams& p, int s) {
  Slot<V> r;
  const int rotated = p.rotary_dim / (2 * V);
  r.turned = s < rotated;
  if (r.turned) {
    r.a = IL && V == 1 ? 2 * s : s * V;
    r.b = IL && V == 1 ? 2 * s + 1 : p.rotary_dim / 2 + s * V;
  } else {
    r.a = p.rotary_dim + (s - rotated) * V;
    r.b = r.a + (p.head_dim - p.rotary_dim + 1) / 2;
    if (r.a >= p.rotary_dim + (p.head_dim - p.rotary_dim + 1) / 2) r.a = r.b = p.head_dim;
  }
  r.on = r.a < p.head_dim;
  r.on_b = r.b < p.head_dim;
  return r;
}

// Element of the head that u_i (side 0) or v_i (side 1) of a slot is.
template <int V, bool IL>
__device__ __forceinline__ int slot_element(const Slot<V>& s, int side, int i) {
  if constexpr (IL && V > 1) {
    const int k = 2 * i + side;
    return k < V ? s.a + k : s.b + k - V;
  }
  return (side ? s.b : s.a) + i;
}

template <typename T, int V, bool IL>
__device__ __forceinline__ void to_pairs(const Raw<T, V>& ra, const Raw<T, V>& rb, Vec<V>& u, Vec<V>& v) {
  float a[V], b[V];
  ra.unpack(a);
  rb.unpack(b);
  if constexpr (IL && V > 1) {
    float x[V], y[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      x[i] = i < V / 2 ? a[2 * i] : b[2 * i - V];
      y[i] = i < V / 2 ? a[2 * i + 1] : b[2 * i + 1 - V];
    }
    u.set(x);
    v.set(y);
  } else {
    u.set(a);
    v.set(b);
  }
}

template <typename T, int V, bool IL>
__device__ __forceinline__ void store_pairs(T* out, const Slot<V>& s, bool live, const Vec<V>& u, const Vec<V>& v) {
  float x[V], y[V];
  u.get(x);
  v.get(y);
  if constexpr (IL && V > 1) {
    float a[V], b[V];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      a[2 * i] = x[i];
      a[2 * i + 1] = y[i];
      b[2 * i] = x[V / 2 + i];
      b[2 * i + 1] = y[V / 2 + i];
    }
    if (live && s.on) store_vec<T, V>(out + s.a, a);
    if (live && s.on_b) store_vec<T, V>(out + s.b, b);
  } else {
    if (live && s.on) store_vec<T, V>(out + s.a, x);
    if (live && s.on_b) store_vec<T, V>(out + s.b, y);
  }
}

// Per-pair values (cosines, sines, norm weights) in shared memory: with 8-element slots, piece k (four
// values) of every slot side by side, so that the lanes' 16-byte reads of one piece are consecutive
// (32 bytes apart they would meet in the same banks two by two).
template <int V>
__device__ __forceinline__ int place_of(int slots, int s, int i) {
  if constexpr (V < 8) return s * V + i;
  else return (i / 4 * slots + s) * 4 + i % 4;
}

// The place of a rotated pair's values.
template <int V, bool IL>
__device__ __forceinline__ int pair_at(const RotaryParams& p, int pair) {
  const int rotated = p.rotary_dim / (2 * V);
  if constexpr (IL && V > 1) {
    const int second = pair >= rotated * (V / 2);  // in the slot's second vector
    const int k = pair - second * rotated * (V / 2);
    return place_of<V>(rotated, k / (V / 2), k % (V / 2) + second * (V / 2));
  }
  return place_of<V>(rotated, pair / V, pair % V);
}

template <int V>
__device__ __forceinline__ void load_pairs(const float* table, int slots, int s, Vec<V>& out) {
  if constexpr (V == 8) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const ulonglong2 u = reinterpret_cast<const ulonglong2*>(table)[k * slots + s];
      out.e[2 * k] = u.x;
      out.e[2 * k + 1] = u.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < Vec<V>::N; ++i) out.e[i] = reinterpret_cast<const typename Vec<V>::E*>(table)[s * Vec<V>::N + i];
  }
}

__device__ __forceinline__ int64_t token_position(const RotaryParams& p, int b, int t) {
  const int64_t at = b * p.ps[0] + t * p.ps[1];
  return p.pos64 ? __ldg(static_cast<const long long*>(p.pos) + at) : __ldg(static_cast<const int32_t*>(p.pos) + at);
}

// A token's angles, formed by its warp: magnitude times cosine, sine and negative sine of each pair.
struct TokenAngles {
  float cos[kRotMaxPairs], sin[kRotMaxPairs], neg_sin[kRotMaxPairs];
};

// `turns`: the block's copy of p.turns (lanes that read different constants wait for one another). FINE (32-bit
// tensors): the part of the angle that its rounding to fp32 lost, at most 1e-7, turns cosine and sine once more, to first order.
template <int V, bool IL, bool FINE>
__device__ __forceinline__ void token_angles(const RotaryParams& p, const uint64_t* turns, int64_t position, int lane,
                                             TokenAngles& out) {
  for (int i = lane; i < p.rotary_dim / 2; i += 32) {
    const uint64_t turn = static_cast<uint64_t>(position) * turns[i];
    float s, c;
    // the top 32 bits as a signed number: units of 2^-31 half turns
    const float top = static_cast<float>(static_cast<int32_t>(turn >> 32));
    sincospif(top * 4.656612873077393e-10f, &s, &c);
    if constexpr (FINE) {
      const uint64_t rest = turn - (static_cast<uint64_t>(static_cast<int64_t>(top)) << 32);  // (modulo a turn)
      const float angle = static_cast<float>(static_cast<int64_t>(rest)) * 3.4061215800865545e-19f;  // 2 pi / 2^64
      const float fine = fmaf(angle, c, s);
      c = fmaf(-angle, s, c);
      s = fine;
    }
    s *= p.magnitude * p.sin_sign;
    const int at = pair_at<V, IL>(p, i);
    out.cos[at] = p.magnitude * c;
    out.sin[at] = s;
    out.neg_sin[at] = -s;
  }
  __syncwarp();
}

// The angles of slot s. A slot that passes through has none: multiplied by (1, 0) instead, an infinity in one
// of its values would become NaN in another.
template <int V>
struct SlotAngles {
  Vec<V> cos, sin, neg_sin;

  __device__ __forceinline__ void load(const RotaryParams& p, const TokenAngles& t, int s) {
    const int rotated = p.rotary_dim / (2 * V);
    load_pairs<V>(t.cos, rotated, s, cos);
    load_pairs<V>(t.sin, rotated, s, sin);
    load_pairs<V>(t.neg_sin, rotated, s, neg_sin);
  }
  __device__ __forceinline__ void turn(Vec<V>& u, Vec<V>& v) const {
#pragma unroll
    for (int i = 0; i < Vec<V>::N; ++i) {
      const auto x = fma_v(u.e[i], cos.e[i], mul_v(v.e[i], neg_sin.e[i]));
      v.e[i] = fma_v(v.e[i], cos.e[i], mul_v(u.e[i], sin.e[i]));
      u.e[i] = x;
    }
  }
};

// The norm weights of a head in pair order, zero outside the head.
struct PairWeights {
  float u[kRotMaxPairs], v[kRotMaxPairs];
};

template <int V, bool IL>
__device__ __forceinline__ void load_pair_weights(const RotaryParams& p, int which, int slots, PairWeights& out) {
  for (int i = threadIdx.x; i < slots * V; i += blockDim.x) {
    const Slot<V> s = slot_of<V, IL>(p, i / V);
    const int eu = slot_element<V, IL>(s, 0, i % V), ev = slot_element<V, IL>(s, 1, i % V);
    out.u[place_of<V>(slots, i / V, i % V)] = eu < p.head_dim ? load_weight(p.w[which], p.w_dtype, eu) : 0.f;
    out.v[place_of<V>(slots, i / V, i % V)] = ev < p.head_dim ? load_weight(p.w[which], p.w_dtype, ev) : 0.f;
  }
}

// Sums over the `lanes` lanes of a head (a power of two, uniform over the grid).
template <int N>
__device__ __forceinline__ void group_sum(float (&v)[N], int lanes) {
#pragma unroll
  for (int o = 16; o > 0; o /= 2) {
    if (lanes > o) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    }
  }
}

// NS: slots of a lane. 32 lanes with one slot each cover 512 elements in 8-element vectors, 128 in pairs and 64
// in single ones; larger heads of the narrow widths take kRotMaxPairs / (32 V) slots, whose unrolled loops
// would cost the small heads up to eight times their work.
template <int V>
constexpr int rotary_most_slots() {
  return kRotMaxPairs / (32 * V);
}

// Both kernels walk units (a token's group of heads) in passes of at_once heads, and fetch the values of
// the next passes, of the next units if need be, while they work on the current one. Four KB a warp are
// on their way at any time: with one pass of register loads ahead (1 KB) the reads stopped at 2.3 TB/s,
// waiting for a memory latency of about 1 us under load. The fetched bytes go to shared memory by
// cp.async, each lane reads back only what it fetched itself, so no lane waits for another.
template <typename T, int V, int VECTORS>  // VECTORS: V-element vectors of a lane in a pass
struct PassRing {
  static constexpr int kBytes = V * static_cast<int>(sizeof(T));
  static constexpr int kPass = VECTORS * 32 * (kBytes < 4 ? 4 : kBytes);
  static constexpr int kStages = kPass >= 2048 ? 2 : kPass >= 1536 ? 3 : 4;
  static constexpr bool kAsync = kBytes >= 4;  // cp.async moves at least 4 bytes
  static constexpr int kWords = kBytes >= 16 ? 4 : kBytes >= 4 ? kBytes / 4 : 1;  // of one access
  static constexpr int kParts = kBytes > 16 ? kBytes / 16 : 1;                    // accesses of a vector
  uint32_t w[kStages][VECTORS][kParts][32][kWords];

  __device__ __forceinline__ void clear(int v, int lane) {
    for (int s = 0; s < kStages; ++s)
      for (int q = 0; q < kParts; ++q)
        for (int k = 0; k < kWords; ++k) w[s][v][q][lane][k] = 0u;
  }
  __device__ __forceinline__ void fetch(int stage, int v, int lane, const T* p) {
#pragma unroll
    for (int q = 0; q < kParts; ++q) {
      uint32_t* dst = w[stage][v][q][lane];
      if constexpr (kBytes >= 16) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                         static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
                     "l"(reinterpret_cast<const uint4*>(p) + q)
                     : "memory");
      } else if constexpr (kAsync) {
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(
                         static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
                     "l"(p), "n"(kBytes)
                     : "memory");
      } else {
        dst[0] = __ldg(reinterpret_cast<const unsigned short*>(p));
      }
    }
  }
  static __device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
  // all but the newest kStages - 1 fetches have arrived
  static __device__ __forceinline__ void wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory"); }
  __device__ __forceinline__ Raw<T, V> get(int stage, int v, int lane) const {
    Raw<T, V> r;
#pragma unroll
    for (int q = 0; q < kParts; ++q) {
      if constexpr (kWords == 4) {
        const uint4 u = *reinterpret_cast<const uint4*>(w[stage][v][q][lane]);
        r.w[4 * q] = u.x; r.w[4 * q + 1] = u.y; r.w[4 * q + 2] = u.z; r.w[4 * q + 3] = u.w;
      } else if constexpr (kWords == 2) {
        const uint2 u = *reinterpret_cast<const uint2*>(w[stage][v][q][lane]);
        r.w[0] = u.x; r.w[1] = u.y;
      } else {
        r.w[0] = w[stage][v][q][lane][0];
      }
    }
    return r;
  }
};

// A place in the walk: the token and the heads [head, end) left of the unit.
struct RotaryCursor {
  uint32_t unit;
  int b, t, head, end;

  __device__ __forceinline__ void begin(const RotaryParams& p, const FastDiv& units, int heads, uint32_t u) {
    unit = u;
    const uint32_t token = fast_div(u, units);
    b = static_cast<int>(fast_div(token, p.seq));
    t = static_cast<int>(token) - b * static_cast<int>(p.seq.d);
    head = static_cast<int>(u - token * units.d) * p.heads_per_unit;
    end = min(heads, head + p.heads_per_unit);
  }
};

__device__ __forceinline__ int64_t unit_position(const RotaryParams& p, const FastDiv& units, uint32_t u) {
  const uint32_t token = fast_div(u, units);
  const int b = static_cast<int>(fast_div(token, p.seq));
  return token_position(p, b, static_cast<int>(token) - b * static_cast<int>(p.seq.d));
}

template <typename T, int V, int NS, bool NORM, bool IL>
__global__ void __launch_bounds__(32 * kRotWarps, 5) rotary_forward_kernel(const __grid_constant__ RotaryParams p) {
  using Ring = PassRing<T, V, 2 * NS>;
  __shared__ __align__(16) Ring ring_all[kRotWarps];
  __shared__ __align__(16) TokenAngles angles_all[kRotWarps];
  __shared__ uint64_t turns[kRotMaxPairs];
  __shared__ __align__(16) PairWeights weights[NORM ? 2 : 1];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  Ring& ring = ring_all[warp];
  TokenAngles& angles = angles_all[warp];
  for (int i = threadIdx.x; i < p.rotary_dim / 2; i += blockDim.x) turns[i] = p.turns[i];
  const int heads = p.heads[0] + p.heads[1];
  const uint32_t total = static_cast<uint32_t>(p.tokens) * p.units[0].d;  // below 2^31: checked by the host
  const uint32_t stride = gridDim.x * kRotWarps;
  const int sub = lane / p.lanes, sl = lane % p.lanes, at_once = 32 / p.lanes;
  const int slots = NS * p.lanes;
  Slot<V> slot[NS];
#pragma unroll
  for (int n = 0; n < NS; ++n) {
    slot[n] = slot_of<V, IL>(p, sl + n * p.lanes);
    // a vector that lies outside the head counts as zeros
    if (!slot[n].on) ring.clear(2 * n, lane);
    if (!slot[n].on_b) ring.clear(2 * n + 1, lane);
  }
  if constexpr (NORM) {
    load_pair_weights<V, IL>(p, 0, slots, weights[0]);
    load_pair_weights<V, IL>(p, 1, slots, weights[1]);
  }
  __syncthreads();
  const uint32_t first = blockIdx.x * kRotWarps + warp;
  if (first >= total) return;

  RotaryCursor in, at;  // of the fetches, of the work
  const T *xq = nullptr, *xk = nullptr;
  bool more_in = true;
  auto begin_in = [&](uint32_t u) {
    in.begin(p, p.units[0], heads, u);
    xq = static_cast<const T*>(p.x[0]) + in.b * p.xs[0][0] + in.t * p.xs[0][1];
    xk = static_cast<const T*>(p.x[1]) + in.b * p.xs[1][0] + in.t * p.xs[1][1];
  };
  auto fetch = [&](int stage) {
    if (more_in) {
      const int h = in.head + sub;
      const bool key = h >= p.heads[0];
      const T* x = (key ? xk : xq) + static_cast<int64_t>(key ? h - p.heads[0] : h) * (key ? p.xh[1] : p.xh[0]);
      if (h < in.end) {  // a lane whose head is behind the unit's keeps older values, which go nowhere
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          if (slot[n].on) ring.fetch(stage, 2 * n, lane, x + slot[n].a);
          if (slot[n].on_b) ring.fetch(stage, 2 * n + 1, lane, x + slot[n].b);
        }
      }
      in.head += at_once;
      if (in.head >= in.end) {
        more_in = in.unit + stride < total;
        if (more_in) begin_in(in.unit + stride);
      }
    }
    Ring::commit();
  };
  begin_in(first);
#pragma unroll
  for (int s = 0; s < Ring::kStages - 1; ++s) fetch(s);
  at.begin(p, p.units[0], heads, first);
  int64_t position = unit_position(p, p.units[0], first);
  SlotAngles<V> sa[NS];
  T *oq = nullptr, *ok = nullptr;
  bool fresh = true;  // the pass is its unit's first
  for (int stage = 0;; stage = stage + 1 == Ring::kStages ? 0 : stage + 1) {
    fetch(stage == 0 ? Ring::kStages - 1 : stage - 1);
    if (fresh) {
      oq = static_cast<T*>(p.out[0]) + at.b * p.os[0][0] + at.t * p.os[0][1];
      ok = static_cast<T*>(p.out[1]) + at.b * p.os[1][0] + at.t * p.os[1][1];
      __syncwarp();  // the previous unit's angles have been read
      token_angles<V, IL, sizeof(T) == 4>(p, turns, position, lane, angles);
#pragma unroll
      for (int n = 0; n < NS; ++n)
        if (slot[n].turned) sa[n].load(p, angles, sl + n * p.lanes);
      // the next unit's position, wanted when this one is done
      if (at.unit + stride < total) position = unit_position(p, p.units[0], at.unit + stride);
    }
    Ring::wait();
    Vec<V> u[NS], v[NS];
#pragma unroll
    for (int n = 0; n < NS; ++n)
      to_pairs<T, V, IL>(ring.get(stage, 2 * n, lane), ring.get(stage, 2 * n + 1, lane), u[n], v[n]);
    const int h = at.head + sub;
    const bool live = h < at.end, key = h >= p.heads[0];
    T* out = (key ? ok : oq) + static_cast<int64_t>(key ? h - p.heads[0] : h) * (key ? p.oh[1] : p.oh[0]);
    typename Vec<V>::E r = Vec<V>::all(1.f);
    if constexpr (NORM) {
      Vec<V> ss;
      ss.fill(0.f);
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int i = 0; i < Vec<V>::N; ++i) ss.e[i] = fma_v(v[n].e[i], v[n].e[i], fma_v(u[n].e[i], u[n].e[i], ss.e[i]));
      float sum[1] = {ss.sum()};
      group_sum(sum, p.lanes);
      r = Vec<V>::all(rsqrtf(sum[0] * p.inv_head_dim + p.eps));
    }
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      if constexpr (NORM) {
        Vec<V> wu, wv;
        load_pairs<V>(weights[key].u, slots, sl + n * p.lanes, wu);
        load_pairs<V>(weights[key].v, slots, sl + n * p.lanes, wv);
#pragma unroll
        for (int i = 0; i < Vec<V>::N; ++i) {
          u[n].e[i] = mul_v(mul_v(u[n].e[i], r), wu.e[i]);
          v[n].e[i] = mul_v(mul_v(v[n].e[i], r), wv.e[i]);
        }
      }
      if (slot[n].turned) sa[n].turn(u[n], v[n]);
      store_pairs<T, V, IL>(out, slot[n], live, u[n], v[n]);
    }
    at.head += at_once;
    fresh = at.head >= at.end;
    if (fresh) {
      if (at.unit + stride >= total) break;
      at.begin(p, p.units[0], heads, at.unit + stride);
    }
  }
}

// Backward of the normed form. Each lane adds up the weight gradients of its elements over every head
// it meets, the block adds its warps' and head groups' sums in a fixed order and writes one partial row;
// norm_weight_grad_kernel adds the blocks' rows, again in a fixed order: the same inputs give the same
// bits. Angles and weights stay in shared memory: in registers they would leave room for half as many
// warps.
template <typename T, int V, int NS, bool IL>
__global__ void __launch_bounds__(32 * kRotWarps, 4)
    qk_norm_rotary_backward_kernel(const __grid_constant__ RotaryParams p) {
  using Ring = PassRing<T, V, 4 * NS>;  // vector 4 n: x's a, + 1: x's b, + 2, + 3: dy's
  union Shared {
    Ring ring[kRotWarps];
    float dw[kRotWarps][ORDA_ROTARY_MAX_DIM];
  };
  __shared__ __align__(16) Shared sh;
  __shared__ __align__(16) TokenAngles angles_all[kRotWarps];
  __shared__ __align__(16) PairWeights weights;
  __shared__ uint64_t turns[kRotMaxPairs];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  Ring& ring = sh.ring[warp];
  TokenAngles& angles = angles_all[warp];
  for (int i = threadIdx.x; i < p.rotary_dim / 2; i += blockDim.x) turns[i] = p.turns[i];
  const uint32_t stride = gridDim.x * kRotWarps, first = blockIdx.x * kRotWarps + warp;
  const int sub = lane / p.lanes, sl = lane % p.lanes, at_once = 32 / p.lanes;
  const int slots = NS * p.lanes;
  Slot<V> slot[NS];
#pragma unroll
  for (int n = 0; n < NS; ++n) slot[n] = slot_of<V, IL>(p, sl + n * p.lanes);
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    __syncthreads();  // the previous weights and sums have been read
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (!slot[n].on) ring.clear(4 * n + 2 * j, lane);
        if (!slot[n].on_b) ring.clear(4 * n + 2 * j + 1, lane);
      }
    load_pair_weights<V, IL>(p, which, slots, weights);
    __syncthreads();
    const uint32_t total = static_cast<uint32_t>(p.tokens) * p.units[which].d;
    Vec<V> dwu[NS], dwv[NS];
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      dwu[n].fill(0.f);
      dwv[n].fill(0.f);
    }
    if (first < total && p.heads[which] > 0) {
      RotaryCursor in, at;
      const T *x = nullptr, *dy = nullptr;
      bool more_in = true;
      auto begin_in = [&](uint32_t u) {
        in.begin(p, p.units[which], p.heads[which], u);
        x = static_cast<const T*>(p.x[which]) + in.b * p.xs[which][0] + in.t * p.xs[which][1];
        dy = static_cast<const T*>(p.dy[which]) + in.b * p.ds[which][0] + in.t * p.ds[which][1];
      };
      auto fetch = [&](int stage) {
        if (more_in) {
          const int h = in.head + sub;
          if (h < in.end) {
            const T* xh = x + static_cast<int64_t>(h) * p.xh[which];
            const T* zh = dy + static_cast<int64_t>(h) * p.dh[which];
#pragma unroll
            for (int n = 0; n < NS; ++n) {
              if (slot[n].on) {
                ring.fetch(stage, 4 * n, lane, xh + slot[n].a);
                ring.fetch(stage, 4 * n + 2, lane, zh + slot[n].a);
              }
              if (slot[n].on_b) {
                ring.fetch(stage, 4 * n + 1, lane, xh + slot[n].b);
                ring.fetch(stage, 4 * n + 3, lane, zh + slot[n].b);
              }
            }
          }
          in.head += at_once;
          if (in.head >= in.end) {
            more_in = in.unit + stride < total;
            if (more_in) begin_in(in.unit + stride);
          }
        }
        Ring::commit();
      };
      begin_in(first);
#pragma unroll
      for (int s = 0; s < Ring::kStages - 1; ++s) fetch(s);
      at.begin(p, p.units[which], p.heads[which], first);
      int64_t position = unit_position(p, p.units[which], first);
      T* out_token = nullptr;
      bool fresh = true;
#pragma unroll 1
      for (int stage = 0;; stage = stage + 1 == Ring::kStages ? 0 : stage + 1) {
        fetch(stage == 0 ? Ring::kStages - 1 : stage - 1);
        if (fresh) {
          out_token = static_cast<T*>(p.out[which]) + at.b * p.os[which][0] + at.t * p.os[which][1];
          __syncwarp();  // the previous unit's angles have been read
          token_angles<V, IL, sizeof(T) == 4>(p, turns, position, lane, angles);
          if (at.unit + stride < total) position = unit_position(p, p.units[which], at.unit + stride);
        }
        Ring::wait();
        Vec<V> u[NS], v[NS], zu[NS], zv[NS];
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          to_pairs<T, V, IL>(ring.get(stage, 4 * n, lane), ring.get(stage, 4 * n + 1, lane), u[n], v[n]);
          to_pairs<T, V, IL>(ring.get(stage, 4 * n + 2, lane), ring.get(stage, 4 * n + 3, lane), zu[n], zv[n]);
        }
        const int h = at.head + sub;
        const bool live = h < at.end;
        T* out = out_token + static_cast<int64_t>(h) * p.oh[which];
        Vec<V> ss, ex;  // sum x^2, sum (w dz) x
        ss.fill(0.f);
        ex.fill(0.f);
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          if (slot[n].turned) {
            SlotAngles<V> sa;
            sa.load(p, angles, sl + n * p.lanes);
            sa.turn(zu[n], zv[n]);
          }
          Vec<V> wu, wv;
          load_pairs<V>(weights.u, slots, sl + n * p.lanes, wu);
          load_pairs<V>(weights.v, slots, sl + n * p.lanes, wv);
#pragma unroll
          for (int i = 0; i < Vec<V>::N; ++i) {
            ss.e[i] = fma_v(v[n].e[i], v[n].e[i], fma_v(u[n].e[i], u[n].e[i], ss.e[i]));
            ex.e[i] = fma_v(mul_v(zu[n].e[i], wu.e[i]), u[n].e[i], ex.e[i]);
            ex.e[i] = fma_v(mul_v(zv[n].e[i], wv.e[i]), v[n].e[i], ex.e[i]);
          }
        }
        float sum[2] = {ss.sum(), ex.sum()};
        group_sum(sum, p.lanes);
        const float r = rsqrtf(sum[0] * p.inv_head_dim + p.eps);
        // -r^2 mean(e n), in an order that leaves a head of zeros 0 where r^3 overflows (eps below 1e-25)
        const float m = -(sum[1] * p.inv_head_dim * r) * r * r;
        const auto r2 = Vec<V>::all(r), m2 = Vec<V>::all(m);
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          Vec<V> wu, wv;
          load_pairs<V>(weights.u, slots, sl + n * p.lanes, wu);
          load_pairs<V>(weights.v, slots, sl + n * p.lanes, wv);
#pragma unroll
          for (int i = 0; i < Vec<V>::N; ++i) {
            const auto tu = mul_v(zu[n].e[i], r2), tv = mul_v(zv[n].e[i], r2);  // r dz
            if (live) {
              dwu[n].e[i] = fma_v(tu, u[n].e[i], dwu[n].e[i]);
              dwv[n].e[i] = fma_v(tv, v[n].e[i], dwv[n].e[i]);
            }
            u[n].e[i] = fma_v(u[n].e[i], m2, mul_v(tu, wu.e[i]));
            v[n].e[i] = fma_v(v[n].e[i], m2, mul_v(tv, wv.e[i]));
          }
          store_pairs<T, V, IL>(out, slot[n], live, u[n], v[n]);
        }
        at.head += at_once;
        fresh = at.head >= at.end;
        if (fresh) {
          if (at.unit + stride >= total) break;
          at.begin(p, p.units[which], p.heads[which], at.unit + stride);
        }
      }
    }
    // head groups of the warp, then the warps of the block
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();  // the sums take the rings' place
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      float du[V], dv[V];
      dwu[n].get(du);
      dwv[n].get(dv);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        for (int o = p.lanes; o < 32; o *= 2) {
          du[i] += __shfl_xor_sync(0xffffffffu, du[i], o);
          dv[i] += __shfl_xor_sync(0xffffffffu, dv[i], o);
        }
        const int eu = slot_element<V, IL>(slot[n], 0, i), ev = slot_element<V, IL>(slot[n], 1, i);
        if (sub == 0 && eu < p.head_dim) sh.dw[warp][eu] = du[i];
        if (sub == 0 && ev < p.head_dim) sh.dw[warp][ev] = dv[i];
      }
    }
    __syncthreads();
    float* row = p.dw_partial + (static_cast<int64_t>(blockIdx.x) * 2 + which) * p.head_dim;
    for (int i = threadIdx.x; i < p.head_dim; i += blockDim.x) {
      float v = 0.f;
#pragma unroll
      for (int k = 0; k < kRotWarps; ++k) v += sh.dw[k][i];
      row[i] = v;
    }
  }
}

// dweight[which][i] = sum over the blocks' partial rows, in a fixed order; one block per kNormSumCols columns of one
// weight, the rows shared out over its threads so that each has its few loads in flight at once (with 32
// columns a block, a warp a row, this took 7 us: five memory latencies).
constexpr int kNormSumCols = 8;

static __global__ void __launch_bounds__(1024) norm_weight_grad_kernel(const float* __restrict__ partial, int rows,
                                                                       int head_dim, int dtype, void* dwq, void* dwk) {
  constexpr int kParts = 1024 / kNormSumCols;
  __shared__ float acc[kNormSumCols][kParts + 1];
  const int which = blockIdx.y, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int c = threadIdx.x % kNormSumCols, part = threadIdx.x / kNormSumCols;
  const int col = blockIdx.x * kNormSumCols + c;
  float v = 0.f;
  if (col < head_dim) {
    constexpr int kBatch = 5;  // all rows of a full grid: 4 x 148
    for (int r = part; r < rows; r += kBatch * kParts) {
      float x[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k)
        x[k] = r + k * kParts < rows ? partial[(static_cast<int64_t>(r + k * kParts) * 2 + which) * head_dim + col] : 0.f;
#pragma unroll
      for (int k = 0; k < kBatch; ++k) v += x[k];
    }
  }
  acc[c][part] = v;
  __syncthreads();
  const int out_col = blockIdx.x * kNormSumCols + warp;
  if (warp >= kNormSumCols || out_col >= head_dim) return;
  v = 0.f;
#pragma unroll
  for (int k = 0; k < kParts / 32; ++k) v += acc[warp][lane + 32 * k];
  for (int o = 16; o > 0; o /= 2) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (lane != 0) return;
  void* out = which ? dwk : dwq;
  if (dtype == ORDA_F32) static_cast<float*>(out)[out_col] = v;
  else if (dtype == ORDA_F16) static_cast<__half*>(out)[out_col] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(out)[out_col] = __float2bfloat16_rn(v);
}

}  // namespace orda
