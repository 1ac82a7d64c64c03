/*
 * orda_b200_student.h - C ABI of the operators around the distillation loss in a student's training
 * step and in its token-by-token run: gated feed-forward block, rotary positions (with or without
 * per-head norms of queries and keys), global gradient norm and clipping.
 *
 * The conventions of orda_b200.h hold: pointers are device pointers owned by the caller unless
 * stated, nothing is allocated and no stream is synchronised, every call only enqueues work on
 * `stream` (a cudaStream_t passed as void*) of the current device, argument errors return an
 * ORDA_ERR_* code before anything is launched, device errors (a pipeline wait that timed out) go to
 * *device_status. The calls keep no state: they may run at the same time from any number of threads,
 * streams and captured graphs as long as their outputs and workspaces differ.
 */
#ifndef ORDA_B200_STUDENT_H_
#define ORDA_B200_STUDENT_H_

#include "orda_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- gated feed-forward block: h = act(x Wgate^T) * (x Wup^T) ---- */
#define ORDA_ACT_SILU 0       /* g / (1 + e^-g)                                             */
#define ORDA_ACT_GELU 1       /* g Phi(g)                                                   */
#define ORDA_ACT_GELU_TANH 2  /* g / 2 (1 + tanh(sqrt(2/pi) (g + 0.044715 g^3)))            */
#define ORDA_ACT_RELU 3       /* max(g, 0), derivative 0 at 0                               */

/* Up to this many rows the 16-bit forward call needs no status word from its caller: a pipeline wait that
   timed out leaves NaN in h. */
#define ORDA_GLU_FEW_ROWS 128

typedef struct orda_glu_args {
  int32_t abi_version;   /* = ORDA_ABI_VERSION */
  int32_t dtype;         /* ORDA_F32 / ORDA_F16 / ORDA_BF16 of every tensor below            */
  int32_t activation;    /* ORDA_ACT_*                                                       */
  int32_t reserved;
  int64_t rows;          /* tokens N                                                         */
  int64_t hidden;        /* H                                                                */
  int64_t ffn;           /* F                                                                */
  const void* x; int64_t ld_x;          /* [N, H]                                            */
  const void* gate; int64_t ld_gate;    /* [F, H]                                            */
  const void* up; int64_t ld_up;        /* [F, H]                                            */
  /* 16-bit types: hidden and the strides of x, gate, up multiples of 8; ld_pre always. Bases 16-byte aligned,
     but for h and dh, which may start at any element.                                      */
  void* h; int64_t ld_h;                /* [N, F]; ld_h is the row stride of dh too          */
  void* pre_gate; int64_t ld_pre;       /* [N, F] x Wgate^T, written where not NULL          */
  void* pre_up;                         /* [N, F] x Wup^T (both or neither)                  */
  /* backward */
  int64_t grad_cols;                    /* columns (and row stride) of dx and dweights: H, or fewer where the
                                           operands' rows end in padding (orda_pad_rows)     */
  const void* dh;                       /* [N, F]                                            */
  void* dx;                             /* [N, grad_cols] or NULL                            */
  void* dweights;                       /* [ceil8(F) + F, grad_cols] or NULL: rows 0 .. F-1 the gradient of
                                           gate, rows ceil8(F) .. that of up; the rows between (at
                                           most 7) hold no value                             */
  int32_t* device_status;               /* int32 device word, zero on entry of a forward call; a backward call
                                           clears it. May be NULL for ORDA_F32 and for a forward call of
                                           at most ORDA_GLU_FEW_ROWS rows. Where it reports a
                                           timeout, the first value of h, dx or of both gradients in
                                           dweights is NaN */
} orda_glu_args_t;

/* Copies of up to three 16-bit matrices (rows of `cols` elements, any alignment, ld[i] elements apart) whose
 * rows end in zeros at a multiple of 8 elements: operands of the calls below with a hidden size that is
 * none. dst[i]: [rows[i], ceil8(cols)], 16-byte aligned. HOST arrays of `count`. */
int32_t orda_pad_rows(int32_t count, const void* const* src, const int64_t* ld, const int64_t* rows, int64_t cols,
                      void* const* dst, void* stream);

/* h (and, where asked for, the products before the activation, which the backward pass reads). */
int32_t orda_glu_forward(const orda_glu_args_t* args, void* stream);
size_t orda_glu_backward_workspace_bytes(const orda_glu_args_t* args);
/* dx = dg Wgate + du Wup, dWgate = dg^T x, dWup = du^T x with dg = dh u act'(g), du = dh act(g);
 * dg and du are rounded to the tensors' type between the two steps. */
int32_t orda_glu_backward(const orda_glu_args_t* args, void* workspace, size_t workspace_bytes, void* stream);

/* ---- rotary positions of queries and keys, alone or after a per-head RMS norm ---- */
#define ORDA_ROTARY_HALF 0         /* pairs (i, i + rotary_dim / 2)                          */
#define ORDA_ROTARY_INTERLEAVED 1  /* pairs (2 i, 2 i + 1)                                   */
#define ORDA_ROTARY_MAX_DIM 512
#define ORDA_ROTARY_MAX_HEADS (1 << 29)

typedef struct orda_rotary_args {
  int32_t abi_version;
  int32_t dtype;                 /* of x, out, dy                                            */
  int64_t batch, seq;            /* tokens: [batch, seq]                                     */
  int32_t heads[2];              /* [0] queries, [1] keys; each <= ORDA_ROTARY_MAX_HEADS     */
  int32_t head_dim;              /* D <= ORDA_ROTARY_MAX_DIM                                 */
  int32_t rotary_dim;            /* even, <= D; the rest of a head is not rotated            */
  int32_t layout;                /* ORDA_ROTARY_*                                            */
  int32_t inverse;               /* 1: rotate by the negative angles                         */
  const void* x[2]; int64_t x_stride[2][3];   /* [batch, seq, heads, D]; element strides of the first three */
  void* out[2]; int64_t out_stride[2][3];
  const void* dy[2]; int64_t dy_stride[2][3]; /* backward of the normed form                 */
  const void* positions; int64_t position_stride[2]; /* [batch, seq] integers                */
  int32_t positions_int64;       /* 1: int64, 0: int32                                       */
  int32_t weight_dtype;
  const uint64_t* turns;         /* HOST: rotary_dim / 2 angles per position, from orda_rotary_turns */
  float magnitude;               /* factor of the rotated values                             */
  float eps;
  const void* weight[2];         /* [D] norm weights, both NULL: no norm                     */
  void* dweight[2];              /* [D] their gradients (weight_dtype)                       */
} orda_rotary_args_t;

/* Angles per position in the kernels' form: out[i] = radians[i] / (2 pi) modulo 1, times 2^64. HOST arrays.
 * ORDA_ERR_INVALID_ARGUMENT where an angle is not finite. */
int32_t orda_rotary_turns(const double* radians, int32_t n, uint64_t* out);

/* out = rotate(x) or rotate(weight * x / sqrt(mean x^2 + eps)). */
int32_t orda_rotary_forward(const orda_rotary_args_t* args, void* stream);
/* Of the normed form: out = gradient of x, dweight = gradients of the weights. (The backward pass of
 * the plain form is orda_rotary_forward on dy with `inverse` set.) */
size_t orda_qk_norm_rotary_backward_workspace_bytes(const orda_rotary_args_t* args);
int32_t orda_qk_norm_rotary_backward(const orda_rotary_args_t* args, void* workspace, size_t workspace_bytes,
                                     void* stream);

/* ---- global norm over many tensors, and clipping ---- */
typedef struct orda_tensor_list {
  int32_t abi_version;
  int32_t count;
  const void* const* src;     /* HOST arrays of `count`: device addresses                    */
  void* const* dst;           /* NULL: norm only; dst[i] == src[i]: in place                 */
  const int64_t* numel;
  const int32_t* dtype;       /* ORDA_F32 / ORDA_F16 / ORDA_BF16, of src[i] and dst[i]       */
} orda_tensor_list_t;

size_t orda_clip_workspace_bytes(const orda_tensor_list_t* list);
/* *norm = sqrt(sum of squares over all tensors), accumulated in 64 bits; with dst,
 * dst[i] = src[i] * min(1, max_norm / (norm + eps)). norm: fp32, device memory. */
int32_t orda_clip_gradients(const orda_tensor_list_t* list, double max_norm, double eps, float* norm,
                            void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* ORDA_B200_STUDENT_H_ */
