// Epilogue of the gated feed-forward block, shared by the pair GEMMs: both products of a feature come out
// of one accumulator row, so one thread forms act(gate) * up and nothing but h (and, for training, the
// two products) goes to memory.
#pragma once

#include "gemm_tc.cuh"
#include "glu_math.cuh"
#include "sm100_ptx.cuh"

namespace orda {

// One 32-row x 64-column piece, one row per lane, from registers through the warp's staging buffer to a
// TMA store. w(q, e): words e = 0..3 of the row's 16-byte chunk q.
template <typename Word>
__device__ __forceinline__ void stage_store_piece(const CUtensorMap* map, uint32_t staging, int64_t y0, int64_t c0,
                                                 int lane, Word&& w) {
  // the previous TMA store of this warp must have read the staging buffer
  if (lane == 0) bulk_wait_read_all();
  __syncwarp();
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const uint32_t addr = staging + static_cast<uint32_t>(lane) * 128u +
                          ((static_cast<uint32_t>(q) ^ static_cast<uint32_t>(lane & 7)) << 4);
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(w(q, 0)), "r"(w(q, 1)), "r"(w(q, 2)),
                 "r"(w(q, 3))
                 : "memory");
  }
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    tma_store_2d(map, staging, static_cast<int32_t>(c0), static_cast<int32_t>(y0));
    bulk_commit_group();
  }
}

// The same piece by plain stores, one row at a time (128 contiguous bytes a warp), for rows that are not 16-byte
// aligned. Two-element words where every row starts on their boundary, single elements otherwise.
template <typename T16, typename Word>
__device__ __forceinline__ void store_piece_rows(T16* out, int64_t ld, int64_t M, int64_t N, uint32_t staging,
                                                 int64_t y0, int64_t c0, int lane, Word&& w) {
  if (lane == 0) bulk_wait_read_all();
  __syncwarp();
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const uint32_t addr = staging + static_cast<uint32_t>(lane) * 128u +
                          ((static_cast<uint32_t>(q) ^ static_cast<uint32_t>(lane & 7)) << 4);
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(w(q, 0)), "r"(w(q, 1)), "r"(w(q, 2)),
                 "r"(w(q, 3))
                 : "memory");
  }
  __syncwarp();
  const int rows = static_cast<int>(M - y0 < 32 ? M - y0 : 32);
  const int64_t col = c0 + 2 * lane;
  const bool words = (ld & 1) == 0 && (reinterpret_cast<uintptr_t>(out) & 3u) == 0 && col + 1 < N;
  for (int r = 0; r < rows; ++r) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];"
                 : "=r"(v)
                 : "r"(staging + static_cast<uint32_t>(r) * 128u +
                       (((static_cast<uint32_t>(lane) >> 2) ^ static_cast<uint32_t>(r & 7)) << 4) + (lane & 3) * 4u)
                 : "memory");
    T16* o = out + (y0 + r) * ld + col;
    if (words) {
      *reinterpret_cast<uint32_t*>(o) = v;
    } else if (col < N) {
      const T16* e = reinterpret_cast<const T16*>(&v);
      o[0] = e[0];
      if (col + 1 < N) o[1] = e[1];
    }
  }
  __syncwarp();  // the rows have been read: the buffer is free again
}

// Gated epilogue of the warp's 32 rows and features [f0 + 64 first, f0 + 64 last) of a 128-feature tile
// (accumulator columns 0..127 gate, 128..255 up): h = act(g) u, and g and u themselves where the backward
// pass will want them, 64 features at a time through the staging buffer.
template <typename T16>
__device__ __forceinline__ void glu_store(const TcGemmParams& p, uint32_t tbase, uint32_t staging, int64_t y0,
                                               int64_t f0, int first, int last, int lane) {
#pragma unroll 1
  for (int half = first; half < last; ++half) {
    const int64_t c0 = f0 + half * 64;
    uint32_t g[2][32], u[2][32];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      tmem_ld32_async(tbase + half * 64 + c * 32, g[c]);
      tmem_ld32_async(tbase + 128 + half * 64 + c * 32, u[c]);
    }
    tmem_wait_ld();
    if (c0 >= p.st.N || y0 >= p.st.M) continue;  // warp-uniform
    auto pair_of = [&](uint32_t (&v)[2][32], int q, int e) {
      const int i = (q & 3) * 8 + 2 * e;
      return pack2<T16>(__uint_as_float(v[q >> 2][i]), __uint_as_float(v[q >> 2][i + 1]));
    };
    if (p.glu_save) {
      stage_store_piece(&p.ws_s_map, staging, y0, c0, lane, [&](int q, int e) { return pair_of(g, q, e); });
      stage_store_piece(&p.ws_t_map, staging, y0, c0, lane, [&](int q, int e) { return pair_of(u, q, e); });
    }
    with_act(p.glu_act, [&](auto tag) {
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          float a, d;
          glu_act<decltype(tag)::kAct, false>(__uint_as_float(g[c][j]), a, d);
          u[c][j] = __float_as_uint(a * __uint_as_float(u[c][j]));
        }
    });
    auto h_word = [&](int q, int e) { return pair_of(u, q, e); };
    if (p.glu_h) store_piece_rows(static_cast<T16*>(p.glu_h), p.st.ldo, p.st.M, p.st.N, staging, y0, c0, lane, h_word);
    else stage_store_piece(&p.out_map, staging, y0, c0, lane, h_word);
  }
}

}  // namespace orda
