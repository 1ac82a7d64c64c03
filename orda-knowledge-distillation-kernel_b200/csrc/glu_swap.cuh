// Gated feed-forward block for a batch of decoded tokens: too many rows for the weight-streaming kernel
// of glu.cuh (its mma.sync fragments re-read x per 16 features), too few to fill the 256-row tiles of the
// pair GEMMs.
//
// The operands change places: the weights are the M side of the tensor-core product, the tokens its N
// side, so a tile costs what its tokens cost. A block multiplies 64 gate rows and the same 64 up rows
// (M = 128: TMEM lanes 0..63 gate, 64..127 up) by all tokens, at most 128; both products meet in shared memory,
// from where the activation and the product go out in whole rows. One tile a block, no persistence: two
// blocks fit an SM, so one's epilogue runs under the other's loads, and 8 stages of weights are on
// their way per SM. What bounds it: reading the weights.
//
// Where the feature tiles alone leave SMs idle, a cluster of blocks shares a tile's K range: every block
// forms its part of the products, then each takes some of the tile's tokens and adds the others' parts
// up through distributed shared memory, in the blocks' order.
//
// Measured in bf16: 64 rows 4096 -> 11264 43 us (4.3 TB/s; the 512-row tiles of the pair GEMM 91, the 256-row
// ones 60), 64 rows 1024 -> 2816 10.3 us with four blocks a tile, 14.4 with one. Short calls are bound by latencies:
// launch and cluster start, the few k blocks of a block, and after them the remote reads, which follow one another
// (each block's `failed`, then each block's part of a token).
//
//   warp 0 : TMA producer    warp 1 : MMA issuer    warps 2..5 : epilogue
//
// The bounded waits' status word lives in shared memory, so that the caller has none to clear; a block
// whose wait runs out flags *status (where the caller gave one) and fills its part of h with NaN.
#pragma once

#include "gemm_tc.cuh"
#include "glu_math.cuh"
#include "sm100_ptx.cuh"

namespace orda {

constexpr int kSwapThreads = 192;
constexpr int kSwapFeatures = 64;
constexpr uint32_t kSwapSmem = 113 * 1024;  // of a block: two fit an SM

struct GluSwapParams {
  CUtensorMap gate, up, x;  // boxes: 64 x 64 of the weights, 64 x tokens of x
  void *h, *pre_gate, *pre_up;
  int64_t ld_h, ld_pre, ffn;
  int32_t rows;
  int32_t tokens;           // tokens of a tile (all rows): a multiple of 16, at most 128
  int32_t stages, kb, kb_part, act;  // k blocks: all, of one block of the cluster
  int32_t split;            // blocks of the cluster
  uint32_t idesc;
  int32_t* status;
};

inline uint32_t swap_stage_bytes(int tokens) { return kATileBytes + static_cast<uint32_t>(tokens) * 128u; }

// from this or another block of the cluster (shared::cluster addresses)
__device__ __forceinline__ float2 cluster_load_float2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ int32_t cluster_load_int(uint32_t addr) {
  int32_t v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

template <typename T16>
__global__ void __launch_bounds__(kSwapThreads, 2) glu_swap_kernel(const __grid_constant__ GluSwapParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[2 * 8 + 1];
  __shared__ int32_t status, failed;
  __shared__ uint32_t tmem_slot;
  const uint32_t tiles = (smem_u32(smem_raw) + 1023u) & ~1023u;
  float* exchange = reinterpret_cast<float*>(smem_raw + (tiles - smem_u32(smem_raw)));
  const uint32_t stage_bytes = kATileBytes + static_cast<uint32_t>(p.tokens) * 128u;
  const uint32_t bar = smem_u32(bars);
  auto full_bar = [&](int s) { return bar + 8u * s; };
  auto empty_bar = [&](int s) { return bar + 8u * (8 + s); };
  const uint32_t done_bar = bar + 8u * 16;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  uint32_t tmem_cols = 32;  // a power of two
  while (tmem_cols < static_cast<uint32_t>(p.tokens)) tmem_cols *= 2;
  const int part = static_cast<int>(blockIdx.x) % p.split;
  const int64_t f0 = (static_cast<int64_t>(blockIdx.x) / p.split) * kSwapFeatures;
  const int kb0 = part * p.kb_part, kbs = min(p.kb_part, p.kb - kb0);  // at least one

  if (threadIdx.x == 0) {
    status = failed = 0;
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    mbar_init(done_bar, 1);
    fence_barrier_init();
    tma_prefetch_desc(&p.gate);
    tma_prefetch_desc(&p.up);
    tma_prefetch_desc(&p.x);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&tmem_slot), tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  bool ok = true;
  if (warp == 0) {
    if (lane == 0) {
      for (int kb = 0; kb < kbs; ++kb) {
        const int s = kb % p.stages;
        if (!mbar_wait(empty_bar(s), ((kb / p.stages) & 1) ^ 1u, &status)) break;
        const uint32_t a = tiles + s * stage_bytes;
        mbar_arrive_expect_tx(full_bar(s), stage_bytes);
        tma_load_2d(a, &p.gate, full_bar(s), (kb0 + kb) * kBK, static_cast<int32_t>(f0));
        tma_load_2d(a + kATileBytes / 2, &p.up, full_bar(s), (kb0 + kb) * kBK, static_cast<int32_t>(f0));
        tma_load_2d(a + kATileBytes, &p.x, full_bar(s), (kb0 + kb) * kBK, 0);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      bool fine = true;
      for (int kb = 0; kb < kbs; ++kb) {
        const int s = kb % p.stages;
        if (!mbar_wait(full_bar(s), (kb / p.stages) & 1, &status)) {
          fine = false;
          break;
        }
        tc_fence_after();
        const uint32_t a = tiles + s * stage_bytes, b = a + kATileBytes;
#pragma unroll
        for (int kk = 0; kk < kBK / 16; ++kk)
          tc_mma_f16(tmem, operand_desc<false>(a, kk), operand_desc<false>(b, kk), p.idesc, (kb | kk) != 0);
        tc_commit(empty_bar(s));
      }
      if (fine) tc_commit(done_bar);
    }
  } else {
    const int quarter = warp & 3;
    ok = mbar_wait(done_bar, 0, &status);
    tc_fence_after();
    // every load has landed and every product has been formed: the stages' memory takes
    // exchange[side][token][feature]
    if (ok) {
      float* mine = exchange + (quarter >> 1) * p.tokens * kSwapFeatures + (quarter & 1) * 32 + lane;
      for (int c = 0; c < p.tokens; c += 32) {
        float v[32];
        tmem_ld32(tmem + (static_cast<uint32_t>(quarter * 32) << 16) + c, v);
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (c + j < p.tokens) mine[(c + j) * kSwapFeatures] = v[j];
      }
    }
    tc_fence_before();
    if (!ok) atomicExch(&failed, 1);
  }
  if (p.split > 1) cluster_sync_all();  // every block's part is in its shared memory
  else __syncthreads();
  if (warp >= 2) {
    ok = ok && failed == 0;
    if (p.split > 1)
      for (int r = 0; r < p.split; ++r) ok = ok && cluster_load_int(map_to_cta(smem_u32(&failed), r)) == 0;
    const uint32_t sg = smem_u32(exchange), su = sg + p.tokens * kSwapFeatures * 4;
    const int64_t f = f0 + 2 * lane;
    const bool pair = f + 1 < p.ffn;
    for (int t = part * 4 + warp - 2; t < p.rows; t += 4 * p.split) {
      if (f >= p.ffn) break;
      const float nan = __int_as_float(0x7fffffff);
      const uint32_t at_pair = (t * kSwapFeatures + 2 * lane) * 4;
      float2 g = make_float2(0.f, 0.f), u = g;
      if (p.split == 1) {
        g = *reinterpret_cast<const float2*>(exchange + t * kSwapFeatures + 2 * lane);
        u = *reinterpret_cast<const float2*>(exchange + (p.tokens + t) * kSwapFeatures + 2 * lane);
      } else for (int r = 0; r < p.split; ++r) {
        const float2 x = cluster_load_float2(map_to_cta(sg + at_pair, r)), y = cluster_load_float2(map_to_cta(su + at_pair, r));
        g.x += x.x; g.y += x.y;
        u.x += y.x; u.y += y.y;
      }
      if (!ok) g = u = make_float2(nan, nan);
      float a0 = 0.f, a1 = 0.f, d;
      with_act(p.act, [&](auto tag) {
        glu_act<decltype(tag)::kAct, false>(g.x, a0, d);
        glu_act<decltype(tag)::kAct, false>(g.y, a1, d);
      });
      if (!ok) a0 = a1 = nan;
      auto put = [&](void* out, int64_t ld, float x, float y) {
        T16* o = static_cast<T16*>(out) + t * ld + f;
        if (pair && (reinterpret_cast<uintptr_t>(o) & 3u) == 0) {
          *reinterpret_cast<uint32_t*>(o) = pack2<T16>(x, y);
        } else {
          o[0] = Conv<T16>::from_f(x);
          if (f + 1 < p.ffn) o[1] = Conv<T16>::from_f(y);
        }
      };
      put(p.h, p.ld_h, a0 * u.x, a1 * u.y);
      if (p.pre_gate) {
        put(p.pre_gate, p.ld_pre, g.x, g.y);
        put(p.pre_up, p.ld_pre, u.x, u.y);
      }
    }
    if (!ok && p.status) atomicCAS(p.status, 0, ORDA_ERR_TIMEOUT);
  }
  tc_fence_before();
  if (p.split > 1) cluster_sync_all();  // the others have read this block's part
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    if (*reinterpret_cast<volatile int32_t*>(&status) != 0) __nanosleep(1000000);  // let in-flight copies land
    tmem_dealloc(tmem, tmem_cols);
  }
}

}  // namespace orda
