// Host side of the gated feed-forward block (include/orda_b200_student.h). Included by orda_abi.cu, whose
// tensor-map and GEMM launch helpers it uses.
#pragma once

#include "glu.cuh"
#include "glu_swap.cuh"
#include "orda_b200_student.h"

namespace {

int64_t round8(int64_t v) { return (v + 7) / 8 * 8; }

int check_glu(const orda_glu_args_t* a, bool backward) {
  if (!a || a->abi_version != ORDA_ABI_VERSION) return ORDA_ERR_INVALID_ARGUMENT;
  if (a->dtype != ORDA_F32 && a->dtype != ORDA_F16 && a->dtype != ORDA_BF16) return ORDA_ERR_INVALID_ARGUMENT;
  if (a->activation < ORDA_ACT_SILU || a->activation > ORDA_ACT_RELU) return ORDA_ERR_INVALID_ARGUMENT;
  if (a->rows < 0 || a->hidden <= 0 || a->ffn <= 0) return ORDA_ERR_INVALID_ARGUMENT;
  if (a->rows > (int64_t(1) << 31) - 1024 || a->hidden > (int64_t(1) << 30) || a->ffn > (int64_t(1) << 30))
    return ORDA_ERR_UNSUPPORTED;  // tile coordinates are 32-bit
  if (a->rows == 0) return ORDA_OK;
  if (!a->x || !a->gate || !a->up) return ORDA_ERR_INVALID_ARGUMENT;
  if (!a->device_status && a->dtype != ORDA_F32 && (backward || a->rows > ORDA_GLU_FEW_ROWS))
    return ORDA_ERR_INVALID_ARGUMENT;
  if (a->ld_x < a->hidden || a->ld_gate < a->hidden || a->ld_up < a->hidden || a->ld_h < a->ffn ||
      ((a->pre_gate || backward) && a->ld_pre < a->ffn))
    return ORDA_ERR_INVALID_ARGUMENT;
  if (backward) {
    if (a->grad_cols < 1 || a->grad_cols > a->hidden) return ORDA_ERR_INVALID_ARGUMENT;
    if (!a->pre_gate || !a->pre_up || !a->dh) return ORDA_ERR_INVALID_ARGUMENT;
  } else if (!a->h || (a->pre_gate == nullptr) != (a->pre_up == nullptr)) {
    return ORDA_ERR_INVALID_ARGUMENT;
  }
  auto off = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; };
  const int64_t unit = a->dtype == ORDA_F32 ? 1 : 8;
  if (a->hidden % unit || a->ld_x % unit || a->ld_gate % unit || a->ld_up % unit ||
      ((a->pre_gate || backward) && a->ld_pre % 8))
    return ORDA_ERR_ALIGNMENT;
  const uintptr_t es = esize(a->dtype);
  if (reinterpret_cast<uintptr_t>(a->h) % es || reinterpret_cast<uintptr_t>(a->dh) % es) return ORDA_ERR_ALIGNMENT;
  if (off(a->x) || off(a->gate) || off(a->up) || off(a->pre_gate) || off(a->pre_up) || off(a->dx) || off(a->dweights))
    return ORDA_ERR_ALIGNMENT;
  if (a->dtype == ORDA_F32 && !backward && !a->pre_gate) return ORDA_ERR_INVALID_ARGUMENT;  // its products need a place
  return ORDA_OK;
}

template <typename T16>
int glu_rows_launch(const orda_glu_args_t* a, cudaStream_t s) {
  GluRowsParams p{};
  p.x = a->x; p.gate = a->gate; p.up = a->up;
  p.h = a->h; p.pre_gate = a->pre_gate; p.pre_up = a->pre_up;
  p.ld_x = a->ld_x; p.ld_gate = a->ld_gate; p.ld_up = a->ld_up; p.ld_h = a->ld_h; p.ld_pre = a->ld_pre;
  p.ffn = a->ffn;
  p.rows = static_cast<int32_t>(a->rows); p.hidden = static_cast<int32_t>(a->hidden); p.act = a->activation;
  const int grid = static_cast<int>(cdiv(a->ffn, kGluFeatures));
  count_launch();
  glu_rows_kernel<T16><<<grid, 32 * kGluWarps, 0, s>>>(p);
  return launch_status();
}

template <typename T16>
int glu_swap_launch(const orda_glu_args_t* a, cudaStream_t s) {
  GluSwapParams p{};
  const int tokens = static_cast<int>(cdiv(a->rows, 16) * 16);  // at most 128: ORDA_GLU_FEW_ROWS
  int rc;
  if ((rc = make_map(&p.gate, a->dtype, a->gate, a->hidden, a->ffn, a->ld_gate, 64, kSwapFeatures))) return rc;
  if ((rc = make_map(&p.up, a->dtype, a->up, a->hidden, a->ffn, a->ld_up, 64, kSwapFeatures))) return rc;
  if ((rc = make_map(&p.x, a->dtype, a->x, a->hidden, a->rows, a->ld_x, 64, static_cast<uint32_t>(tokens)))) return rc;
  p.h = a->h; p.pre_gate = a->pre_gate; p.pre_up = a->pre_up;
  p.ld_h = a->ld_h; p.ld_pre = a->ld_pre; p.ffn = a->ffn; p.rows = static_cast<int32_t>(a->rows);
  p.tokens = tokens;
  p.kb = static_cast<int32_t>(cdiv(a->hidden, kBK));
  p.act = a->activation;
  p.idesc = make_idesc_f16(a->dtype == ORDA_BF16 ? 1u : 0u, 128, static_cast<uint32_t>(tokens), 0u, 0u);
  p.status = a->device_status;
  // as many stages as half an SM holds (6 at 16 tokens, 3 at 128); the exchange of the two products needs
  // 512 bytes a token of the same memory
  p.stages = static_cast<int32_t>(std::min<uint32_t>(8, (kSwapSmem - 1024) / swap_stage_bytes(tokens)));
  const uint32_t smem = 1024 + p.stages * swap_stage_bytes(tokens);
  set_smem(glu_swap_kernel<T16>, smem);
  // Blocks that share a tile's K: as many as fit beside the other tiles, two blocks an SM, each with at least
  // four k blocks (one round of stages).
  const int64_t f_tiles = cdiv(a->ffn, kSwapFeatures);
  int64_t split = std::min<int64_t>({8, 2 * num_sms() / f_tiles, p.kb / 4});
  split = std::max<int64_t>(split, 1);
  p.kb_part = static_cast<int32_t>(cdiv(p.kb, split));
  p.split = static_cast<int32_t>(cdiv(p.kb, p.kb_part));  // no block without a k block
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(f_tiles * p.split));
  cfg.blockDim = dim3(kSwapThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute cluster{};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = static_cast<unsigned>(p.split);
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  cfg.attrs = &cluster;
  cfg.numAttrs = 1;
  count_launch();
  cudaLaunchKernelEx(&cfg, glu_swap_kernel<T16>, p);
  return launch_status();
}

// Testing hook (orda_debug_glu_*_marked): every product of the thread's calls ends as if a wait had timed out.
thread_local bool t_mark_products = false;

__global__ void mark_timeout_kernel(const __grid_constant__ TcGemmParams p) { mark_timeout(p); }

int mark_if_testing(const TcGemmParams& prm, cudaStream_t s) {
  if (!t_mark_products) return ORDA_OK;
  mark_timeout_kernel<<<1, 1, 0, s>>>(prm);
  return launch_status();
}

template <typename T16>
int glu_forward_tc(const orda_glu_args_t* a, cudaStream_t s) {
  if (a->rows <= 8) return glu_rows_launch<T16>(a, s);
  if (a->rows <= ORDA_GLU_FEW_ROWS) return glu_swap_launch<T16>(a, s);
  TcGemmParams prm{};
  prm.status = a->device_status;
  int rc;
  if ((rc = make_operand_map(&prm.a0, a->dtype, a->x, false, a->rows, a->hidden, a->ld_x, kTileRows))) return rc;
  if ((rc = make_operand_map(&prm.b0, a->dtype, a->gate, false, a->ffn, a->hidden, a->ld_gate, 128))) return rc;
  if ((rc = make_operand_map(&prm.b1, a->dtype, a->up, false, a->ffn, a->hidden, a->ld_up, 128))) return rc;
  if (a->ld_h % 8 == 0 && (reinterpret_cast<uintptr_t>(a->h) & 15u) == 0) {
    if ((rc = make_map(&prm.out_map, a->dtype, a->h, a->ffn, a->rows, a->ld_h, 64, 32))) return rc;
  } else {
    prm.glu_h = a->h;
    prm.st.ldo = a->ld_h;
  }
  prm.poison[0] = static_cast<uint16_t*>(a->h);
  prm.glu_act = a->activation;
  prm.glu_save = a->pre_gate != nullptr;
  if (prm.glu_save) {
    if ((rc = make_map(&prm.ws_s_map, a->dtype, a->pre_gate, a->ffn, a->rows, a->ld_pre, 64, 32))) return rc;
    if ((rc = make_map(&prm.ws_t_map, a->dtype, a->pre_up, a->ffn, a->rows, a->ld_pre, 64, 32))) return rc;
  }
  prm.kb0 = static_cast<int32_t>(cdiv(a->hidden, kBK));
  prm.st.M = a->rows;
  prm.st.N = a->ffn;
  // 512 x 128 or 256 x 128 tiles: the wide kernel moves a quarter less per product, the 256-row one has two
  // accumulator buffers, so that a short K does not wait for the epilogue, and wastes less of a ragged
  // batch. Estimated clocks of a CTA pair, fitted to K = 1024 ... 4096: 1050 a k block + 9500 a tile against
  // 620 + 2000. (8192 rows, us wide and 256-row: 1024 -> 2816 94 and 82, 1536 -> 4224 181 and 170, 2048 -> 5632
  // 284 and 291, 4096 -> 11264 1036 and 1077.)
  const int64_t pairs = std::max(1, num_sms() / 2), f_tiles = cdiv(a->ffn, 128);
  const int64_t wide = cdiv(cdiv(a->rows, 512) * f_tiles, pairs) * (1050 * prm.kb0 + 9500);
  const int64_t half = cdiv(cdiv(a->rows, 256) * f_tiles, pairs) * (620 * prm.kb0 + 2000);
  const int64_t cols = 2 * round8(a->ffn);
  rc = half < wide ? launch_tc2<false, false, A_PLAIN, false, EPI_GLU, T16>(prm, cdiv(a->rows, 256), cols, s, 8)
                   : launch_tc2w<false, false, A_PLAIN, false, EPI_GLU, T16>(prm, cdiv(a->rows, 512), cols, s, 8);
  return rc ? rc : mark_if_testing(prm, s);
}

// K split of a gradient GEMM with M x N outputs and `kb` k blocks on the wide kernel: the split whose
// estimated time is smallest. A wave (every CTA pair one tile) takes 0.65 us a k block and 4 us more; a
// split adds a launch and the traffic of the fp32 partials, written once and read once at 6.5 TB/s.
int glu_split(int64_t M, int64_t N, int64_t kb) {
  const int64_t tiles = cdiv(M, 512) * cdiv(N, kPairBN);
  const int64_t pairs = std::max(1, num_sms() / 2);
  int best = 1;
  double best_us = 0;
  for (int sp = 1; sp <= 8 && sp <= kb; ++sp) {
    if (sp > 1 && cdiv(kb, sp) * (sp - 1) >= kb) continue;  // a range would be empty
    double us = static_cast<double>(cdiv(tiles * sp, pairs)) * (0.65 * cdiv(kb, sp) + 4.0);
    if (sp > 1) us += 2.5 + (4.0 * sp + 2.0) * M * N / 6.5e6;
    if (sp == 1 || us < best_us) {
      best = sp;
      best_us = us;
    }
  }
  return best;
}

struct GluPlan {
  int64_t fp;             // columns of dg (du follows): ffn rounded up to 8
  int split_dx, split_dw;
  size_t off_part, total;  // dg | du at 0
};

GluPlan plan_glu_backward(const orda_glu_args_t* a) {
  GluPlan p{};
  p.fp = round8(a->ffn);
  p.split_dx = p.split_dw = 1;
  size_t off = align256(esize(a->dtype) * 2 * p.fp * a->rows);
  p.off_part = off;
  if (a->dtype != ORDA_F32) {
    size_t part = 0;
    if (a->dx) {
      p.split_dx = glu_split(a->rows, a->grad_cols, 2 * cdiv(a->ffn, kBK));
      if (p.split_dx > 1) part = std::max(part, sizeof(float) * p.split_dx * a->rows * round8(a->grad_cols));
    }
    if (a->dweights) {
      p.split_dw = glu_split(p.fp + a->ffn, a->grad_cols, cdiv(a->rows, kBK));
      if (p.split_dw > 1)
        part = std::max(part, sizeof(float) * p.split_dw * (p.fp + a->ffn) * round8(a->grad_cols));
    }
    off = align256(off + part);
  }
  p.total = off;
  return p;
}

// [split, M, N] fp32 array in boxes of one split's 32 x 32 values, 128-byte swizzle.
int make_partial_map(CUtensorMap* m, void* base, int64_t N, int64_t M, int split) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return ORDA_ERR_CUDA;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(N), static_cast<cuuint64_t>(M), static_cast<cuuint64_t>(split)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(N) * 4, static_cast<cuuint64_t>(N) * M * 4};
  const cuuint32_t box[3] = {32, 32, 1}, ones[3] = {1, 1, 1};
  const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, base, dims, strides, box, ones,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? ORDA_OK : ORDA_ERR_INVALID_ARGUMENT;
}

// Destination of a gradient GEMM: `out` itself, or fp32 partials added in a fixed order by sum_split_kernel;
// both leave by TMA stores. `second`: the row where another result starts (0: none), marked of its own on a timeout.
template <bool A_MN, bool TWO_SEG, typename T16>
int glu_grad_gemm(TcGemmParams& prm, int dtype, int64_t M, int64_t N, int64_t second, int split, void* out,
                  uint8_t* part, cudaStream_t s) {
  int rc;
  const int64_t np = round8(N);
  for (int i = 0; i < (second ? 2 : 1); ++i)
    prm.poison[i] = split <= 1 ? static_cast<uint16_t*>(out) + i * second * N
                               : reinterpret_cast<uint16_t*>(part) + 2 * i * second * np + 1;
  if (split <= 1) {
    prm.st = StoreEpiParams{out, N, M, N, 0, 0};
    if (N == np) {
      if ((rc = make_map(&prm.out_map, dtype, out, N, M, N, 64, 32))) return rc;  // (clips a last piece at N)
      prm.st_tma = 1;
    } else {
      prm.st_tma = 3;
    }
    rc = launch_tc2w<A_MN, true, A_PLAIN, TWO_SEG, EPI_STORE, T16>(prm, cdiv(M, 512), N, s, 4);
    return rc ? rc : mark_if_testing(prm, s);
  }
  prm.ksplit = split;
  prm.kb_split = static_cast<int32_t>(cdiv(prm.kb0 + prm.kb1, split));
  prm.split_bytes = static_cast<int64_t>(sizeof(float)) * M * np;
  prm.st = StoreEpiParams{part, np, M, np, 1, 0};
  if ((rc = make_partial_map(&prm.out_map, part, np, M, split))) return rc;  // (rows of 32-byte multiples)
  prm.st_tma = 2;
  if ((rc = launch_tc2w<A_MN, true, A_PLAIN, TWO_SEG, EPI_STORE, T16>(prm, cdiv(M, 512), N, s, 4))) return rc;
  if ((rc = mark_if_testing(prm, s))) return rc;
  count_launch();
  const float* sums = reinterpret_cast<const float*>(part);
  if (N == np) {
    const int64_t count8 = M * N / 8;
    sum_split_kernel<T16><<<static_cast<int>(std::min<int64_t>(cdiv(count8, 256), 8 * num_sms())), 256, 0, s>>>(
        sums, split, M * N, static_cast<T16*>(out), count8);
  } else {
    sum_split_rows_kernel<T16><<<static_cast<int>(std::min<int64_t>(cdiv(M * N, 256), 16 * num_sms())), 256, 0, s>>>(
        sums, split, M, N, np, static_cast<T16*>(out));
  }
  return launch_status();
}

template <typename T>
int glu_grad_launch(const orda_glu_args_t* a, const GluPlan& P, T* out, cudaStream_t s) {
  const int64_t vecs = a->rows * (P.fp / 8);
  const int grid = static_cast<int>(std::min<int64_t>(cdiv(vecs, 256), 16 * num_sms()));
  count_launch();
  const bool dh_vec = a->ffn % 8 == 0 && (a->ld_h * sizeof(T)) % 16 == 0 && (reinterpret_cast<uintptr_t>(a->dh) & 15u) == 0;
  glu_grad_kernel<T><<<grid, 256, 0, s>>>(static_cast<const T*>(a->dh), a->ld_h, dh_vec,
                                          static_cast<const T*>(a->pre_gate), static_cast<const T*>(a->pre_up), out,
                                          a->rows, a->ffn, P.fp, a->ld_pre, a->activation, a->device_status,
                                          GluSources{a->x, a->gate, a->up, a->ld_x, a->ld_gate, a->ld_up, a->hidden});
  return launch_status();
}

template <typename T16>
int glu_backward_tc(const orda_glu_args_t* a, const GluPlan& P, uint8_t* ws, cudaStream_t s) {
  T16* dgu = reinterpret_cast<T16*>(ws);
  uint8_t* part = ws + P.off_part;
  const int64_t ld = 2 * P.fp;
  int rc;
  if ((rc = glu_grad_launch<T16>(a, P, dgu, s))) return rc;
  if (a->dx) {  // [dg | du] [Wgate; Wup]: two K segments
    TcGemmParams prm{};
    prm.status = a->device_status;
    if ((rc = make_operand_map(&prm.a0, a->dtype, dgu, false, a->rows, a->ffn, ld, kTileRows))) return rc;
    if ((rc = make_operand_map(&prm.a1, a->dtype, dgu + P.fp, false, a->rows, a->ffn, ld, kTileRows))) return rc;
    if ((rc = make_operand_map(&prm.b0, a->dtype, a->gate, true, a->grad_cols, a->ffn, a->ld_gate, 128))) return rc;
    if ((rc = make_operand_map(&prm.b1, a->dtype, a->up, true, a->grad_cols, a->ffn, a->ld_up, 128))) return rc;
    prm.kb0 = prm.kb1 = static_cast<int32_t>(cdiv(a->ffn, kBK));
    if ((rc = glu_grad_gemm<false, true, T16>(prm, a->dtype, a->rows, a->grad_cols, 0, P.split_dx, a->dx, part, s)))
      return rc;
  }
  if (a->dweights) {  // [dg | du]^T x: both weights' gradients are one product of fp + ffn rows
    TcGemmParams prm{};
    prm.status = a->device_status;
    const int64_t m = P.fp + a->ffn;
    if ((rc = make_operand_map(&prm.a0, a->dtype, dgu, true, m, a->rows, ld, kTileRows))) return rc;
    if ((rc = make_operand_map(&prm.b0, a->dtype, a->x, true, a->grad_cols, a->rows, a->ld_x, 128))) return rc;
    prm.kb0 = static_cast<int32_t>(cdiv(a->rows, kBK));
    if ((rc = glu_grad_gemm<true, false, T16>(prm, a->dtype, m, a->grad_cols, P.fp, P.split_dw, a->dweights, part, s)))
      return rc;
  }
  return ORDA_OK;
}

int glu_forward_f32(const orda_glu_args_t* a, cudaStream_t s) {
  float* g = static_cast<float*>(a->pre_gate);
  float* u = static_cast<float*>(a->pre_up);
  const float* x = static_cast<const float*>(a->x);
  simt_gemm(x, a->ld_x, 1, static_cast<const float*>(a->gate), a->ld_gate, 1, g, a->ld_pre, a->rows, a->ffn, a->hidden, 0, s);
  simt_gemm(x, a->ld_x, 1, static_cast<const float*>(a->up), a->ld_up, 1, u, a->ld_pre, a->rows, a->ffn, a->hidden, 0, s);
  count_launch();
  glu_act_kernel<<<static_cast<int>(std::min<int64_t>(cdiv(a->rows * a->ffn, 256), 16 * num_sms())), 256, 0, s>>>(
      g, u, static_cast<float*>(a->h), a->rows, a->ffn, a->ld_pre, a->ld_h, a->activation);
  return launch_status();
}

int glu_backward_f32(const orda_glu_args_t* a, const GluPlan& P, uint8_t* ws, cudaStream_t s) {
  float* dgu = reinterpret_cast<float*>(ws);
  const int64_t ld = 2 * P.fp;
  const int rc = glu_grad_launch<float>(a, P, dgu, s);
  if (rc) return rc;
  const float* x = static_cast<const float*>(a->x);
  if (a->dx) {
    float* dx = static_cast<float*>(a->dx);
    simt_gemm(dgu, ld, 1, static_cast<const float*>(a->gate), 1, a->ld_gate, dx, a->grad_cols, a->rows, a->grad_cols, a->ffn, 0, s);
    simt_gemm(dgu + P.fp, ld, 1, static_cast<const float*>(a->up), 1, a->ld_up, dx, a->grad_cols, a->rows, a->grad_cols, a->ffn, 1, s);
  }
  if (a->dweights) {
    float* dw = static_cast<float*>(a->dweights);
    simt_gemm(dgu, 1, ld, x, 1, a->ld_x, dw, a->grad_cols, P.fp + a->ffn, a->grad_cols, a->rows, 0, s);
  }
  return launch_status();
}

}  // namespace

extern "C" {

int32_t orda_pad_rows(int32_t count, const void* const* src, const int64_t* ld, const int64_t* rows, int64_t cols,
                      void* const* dst, void* stream) {
  if (count < 0 || count > 3 || cols < 1) return ORDA_ERR_INVALID_ARGUMENT;
  if (count > 0 && (!src || !ld || !rows || !dst)) return ORDA_ERR_INVALID_ARGUMENT;
  PadRowsParams p{};
  p.cols = cols;
  p.cols_pad = round8(cols);
  int64_t total = 0;
  for (int i = 0; i < count; ++i) {
    if (rows[i] < 0 || (rows[i] > 0 && (!src[i] || !dst[i] || ld[i] < 0))) return ORDA_ERR_INVALID_ARGUMENT;
    if ((reinterpret_cast<uintptr_t>(src[i]) & 1u) || (reinterpret_cast<uintptr_t>(dst[i]) & 15u))
      return ORDA_ERR_ALIGNMENT;
    p.src[i] = static_cast<const uint16_t*>(src[i]);
    p.dst[i] = static_cast<uint16_t*>(dst[i]);
    p.ld[i] = ld[i];
    p.last[i] = total += rows[i] * (p.cols_pad / 8);
  }
  if (total == 0) return ORDA_OK;
  p.count = count;
  count_launch();
  pad_rows_kernel<<<static_cast<int>(std::min<int64_t>(cdiv(total, 256), 16 * num_sms())), 256, 0,
                    static_cast<cudaStream_t>(stream)>>>(p);
  return launch_status();
}

int32_t orda_glu_forward(const orda_glu_args_t* args, void* stream) {
  const int rc = check_glu(args, false);
  if (rc || args->rows == 0) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (args->dtype) {
    case ORDA_BF16: return glu_forward_tc<__nv_bfloat16>(args, s);
    case ORDA_F16: return glu_forward_tc<__half>(args, s);
    default: return glu_forward_f32(args, s);
  }
}

size_t orda_glu_backward_workspace_bytes(const orda_glu_args_t* args) {
  if (check_glu(args, true) != ORDA_OK || args->rows == 0) return 0;
  return plan_glu_backward(args).total;
}

int32_t orda_glu_backward(const orda_glu_args_t* args, void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = check_glu(args, true);
  if (rc) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (args->rows == 0) {
    if (args->dweights)
      cudaMemsetAsync(args->dweights, 0, esize(args->dtype) * (round8(args->ffn) + args->ffn) * args->grad_cols, s);
    return launch_status();
  }
  const GluPlan P = plan_glu_backward(args);
  if (!workspace || workspace_bytes < P.total) return ORDA_ERR_WORKSPACE;
  if ((reinterpret_cast<uintptr_t>(workspace) & 15u) != 0) return ORDA_ERR_ALIGNMENT;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  switch (args->dtype) {
    case ORDA_BF16: return glu_backward_tc<__nv_bfloat16>(args, P, ws, s);
    case ORDA_F16: return glu_backward_tc<__half>(args, P, ws, s);
    default: return glu_backward_f32(args, P, ws, s);
  }
}

int32_t orda_debug_glu_forward_marked(const orda_glu_args_t* args, void* stream) {
  t_mark_products = true;
  const int32_t rc = orda_glu_forward(args, stream);
  t_mark_products = false;
  return rc;
}

int32_t orda_debug_glu_backward_marked(const orda_glu_args_t* args, void* workspace, size_t workspace_bytes, void* stream) {
  t_mark_products = true;
  const int32_t rc = orda_glu_backward(args, workspace, workspace_bytes, stream);
  t_mark_products = false;
  return rc;
}

}  // extern "C"
