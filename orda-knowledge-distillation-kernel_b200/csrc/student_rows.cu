// Host side of the memory-bound operators of include/orda_b200_student.h: rotary positions, per-head
// query/key norms and gradient clipping.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "grad_norm.cuh"
#include "host_common.cuh"
#include "orda_b200_student.h"
#include "rotary.cuh"

using namespace orda;

namespace {

bool float_dtype(int32_t d) { return d == ORDA_F32 || d == ORDA_F16 || d == ORDA_BF16; }

// ------------------------------------------------------------------ rotary
int check_rotary(const orda_rotary_args_t* a, bool backward) {
  if (!a || a->abi_version != ORDA_ABI_VERSION || !float_dtype(a->dtype)) return ORDA_ERR_INVALID_ARGUMENT;
  if (a->batch < 0 || a->seq < 0 || a->heads[0] < 0 || a->heads[1] < 0) return ORDA_ERR_INVALID_ARGUMENT;
  if (a->head_dim < 1 || a->rotary_dim < 0 || a->rotary_dim % 2 || a->rotary_dim > a->head_dim)
    return ORDA_ERR_INVALID_ARGUMENT;
  // the kernels count units (a token's groups of heads) and heads and step from head to head in 32 bits
  if (a->head_dim > ORDA_ROTARY_MAX_DIM || a->heads[0] > ORDA_ROTARY_MAX_HEADS || a->heads[1] > ORDA_ROTARY_MAX_HEADS || a->batch > INT32_MAX || a->seq > INT32_MAX ||
      a->batch * a->seq > INT32_MAX)
    return ORDA_ERR_UNSUPPORTED;
  for (int i = 0; i < 2; ++i)
    for (int64_t stride : {a->x_stride[i][2], a->out_stride[i][2], a->dy_stride[i][2]})
      if (stride > INT32_MAX || stride < INT32_MIN) return ORDA_ERR_UNSUPPORTED;
  if (a->layout != ORDA_ROTARY_HALF && a->layout != ORDA_ROTARY_INTERLEAVED) return ORDA_ERR_INVALID_ARGUMENT;
  const bool norm = a->weight[0] || a->weight[1];
  if ((norm || backward) && (!a->weight[0] || !a->weight[1] || !float_dtype(a->weight_dtype)))
    return ORDA_ERR_INVALID_ARGUMENT;
  if (backward && (!a->dweight[0] || !a->dweight[1])) return ORDA_ERR_INVALID_ARGUMENT;
  if (a->batch * a->seq > 0) {
    if (!a->positions || (a->rotary_dim > 0 && !a->turns)) return ORDA_ERR_INVALID_ARGUMENT;
    for (int i = 0; i < 2; ++i)
      if (a->heads[i] > 0 && (!a->x[i] || !a->out[i] || (backward && !a->dy[i]))) return ORDA_ERR_INVALID_ARGUMENT;
  }
  auto off = [](const void* p, size_t element) { return reinterpret_cast<uintptr_t>(p) % element != 0; };
  const size_t es = esize(a->dtype), ws = norm || backward ? esize(a->weight_dtype) : 1;
  if (off(a->positions, a->positions_int64 ? 8 : 4)) return ORDA_ERR_ALIGNMENT;
  for (int i = 0; i < 2; ++i)
    if (off(a->x[i], es) || off(a->out[i], es) || off(a->weight[i], ws) ||
        (backward && (off(a->dy[i], es) || off(a->dweight[i], ws))))
      return ORDA_ERR_ALIGNMENT;
  return ORDA_OK;
}

// Vector width in elements: 8 where every head starts on a 16-byte boundary and both parts of a head
// (rotated, passed through) are whole numbers of 16-element slots; 2 with the same rule for 4-element
// slots and two-element boundaries; else single elements.
int rotary_width(const orda_rotary_args_t* a, bool backward) {
  const size_t es = esize(a->dtype);
  for (int v : {8, 2}) {
    if (a->head_dim % (2 * v) || a->rotary_dim % (2 * v)) continue;
    const uintptr_t bytes = std::min<size_t>(16, v * es);
    const int64_t elems = static_cast<int64_t>(bytes / es);
    bool ok = true;
    auto check = [&](const void* p, const int64_t* st) {
      ok = ok && reinterpret_cast<uintptr_t>(p) % bytes == 0 && st[0] % elems == 0 && st[1] % elems == 0 &&
           st[2] % elems == 0;
    };
    for (int i = 0; i < 2; ++i) {
      if (a->heads[i] == 0) continue;
      check(a->x[i], a->x_stride[i]);
      check(a->out[i], a->out_stride[i]);
      if (backward) check(a->dy[i], a->dy_stride[i]);
    }
    if (ok) return v;
  }
  return 1;
}

struct RotaryPlan {
  RotaryParams p;
  int width, grid;
  bool interleaved, one_slot;  // one_slot: a head's slots fit the 32 lanes
};

// A unit of work (one warp) is a group of heads of one token. Large calls give a warp all heads of a
// token, so that its angles are computed once; calls with fewer tokens than the card has warp slots
// split a token's heads over warps, down to the heads that one warp takes at once.
RotaryPlan plan_rotary(const orda_rotary_args_t* a, bool backward) {
  RotaryPlan r{};
  RotaryParams& p = r.p;
  r.width = rotary_width(a, backward);
  for (int i = 0; i < 2; ++i) {
    p.x[i] = a->x[i]; p.dy[i] = a->dy[i]; p.out[i] = a->out[i]; p.w[i] = a->weight[i];
    for (int j = 0; j < 2; ++j) {
      p.xs[i][j] = a->x_stride[i][j];
      p.os[i][j] = a->out_stride[i][j];
      p.ds[i][j] = a->dy_stride[i][j];
    }
    p.xh[i] = static_cast<int32_t>(a->x_stride[i][2]);
    p.oh[i] = static_cast<int32_t>(a->out_stride[i][2]);
    p.dh[i] = static_cast<int32_t>(a->dy_stride[i][2]);
    p.heads[i] = a->heads[i];
  }
  p.pos = a->positions;
  p.ps[0] = a->position_stride[0]; p.ps[1] = a->position_stride[1];
  p.pos64 = a->positions_int64;
  p.seq = make_fast_div(static_cast<uint32_t>(a->seq));
  p.tokens = static_cast<int32_t>(a->batch * a->seq);
  p.head_dim = a->head_dim; p.rotary_dim = a->rotary_dim;
  r.interleaved = a->layout == ORDA_ROTARY_INTERLEAVED;
  p.inv_head_dim = 1.f / static_cast<float>(a->head_dim);
  p.w_dtype = a->weight_dtype;
  p.magnitude = a->magnitude;
  p.sin_sign = (a->inverse != 0) != backward ? -1.f : 1.f;
  p.eps = a->eps;
  for (int i = 0; i < a->rotary_dim / 2; ++i) p.turns[i] = a->turns[i];
  const int slots = static_cast<int>(cdiv(a->head_dim, 2 * r.width));
  r.one_slot = slots <= 32;
  p.lanes = 1;
  while (p.lanes < slots && p.lanes < 32) p.lanes *= 2;
  const int at_once = 32 / p.lanes;
  const int64_t want = 16 * num_sms();  // warps
  const int first = backward ? a->heads[0] : a->heads[0] + a->heads[1], second = backward ? a->heads[1] : 0;
  int hpu = static_cast<int>(cdiv(std::max({first, second, 1}), at_once)) * at_once;
  // (a unit index stays below 2^31)
  while (hpu > at_once && static_cast<int64_t>(p.tokens) * (cdiv(first, hpu) + cdiv(second, hpu)) < want)
    hpu = static_cast<int>(cdiv(hpu / at_once, 2)) * at_once;
  p.heads_per_unit = hpu;
  const int64_t u0 = cdiv(first, hpu), u1 = cdiv(second, hpu);
  p.units[0] = make_fast_div(static_cast<uint32_t>(std::max<int64_t>(u0, 1)));
  p.units[1] = make_fast_div(static_cast<uint32_t>(std::max<int64_t>(u1, 1)));
  const int64_t units = static_cast<int64_t>(p.tokens) * std::max<int64_t>(u0, u1);
  // no more blocks than run at once (the kernels' launch bounds): a warp walks the units that are left
  r.grid = static_cast<int>(std::min<int64_t>(cdiv(units, kRotWarps), (backward ? 4 : 5) * num_sms()));
  return r;
}

// f(V, NS, IL) of the plan as integral constants. (Single-element slots hold (u, v) in either layout: slot_of
// alone tells the layouts apart.)
template <typename F>
void with_rotary_shape(const RotaryPlan& r, F&& f) {
  auto layout = [&](auto v, auto ns) {
    if (r.interleaved) f(v, ns, std::true_type{});
    else f(v, ns, std::false_type{});
  };
  auto slots = [&](auto v) {
    constexpr int most = rotary_most_slots<decltype(v)::value>();
    if constexpr (most > 1) {
      if (r.one_slot) return layout(v, std::integral_constant<int, 1>{});
    }
    layout(v, std::integral_constant<int, most>{});
  };
  if (r.width == 8) slots(std::integral_constant<int, 8>{});
  else if (r.width == 2) slots(std::integral_constant<int, 2>{});
  else slots(std::integral_constant<int, 1>{});
}

template <typename T>
int dispatch_rotary(const RotaryPlan& r, bool norm, cudaStream_t s) {
  count_launch();
  with_rotary_shape(r, [&](auto v, auto ns, auto il) {
    constexpr int V = decltype(v)::value, NS = decltype(ns)::value;
    constexpr bool IL = decltype(il)::value;
    if (norm) rotary_forward_kernel<T, V, NS, true, IL><<<r.grid, 32 * kRotWarps, 0, s>>>(r.p);
    else rotary_forward_kernel<T, V, NS, false, IL><<<r.grid, 32 * kRotWarps, 0, s>>>(r.p);
  });
  return launch_status();
}

template <typename T>
int dispatch_norm_backward(const RotaryPlan& r, cudaStream_t s) {
  count_launch();
  with_rotary_shape(r, [&](auto v, auto ns, auto il) {
    qk_norm_rotary_backward_kernel<T, decltype(v)::value, decltype(ns)::value, decltype(il)::value>
        <<<r.grid, 32 * kRotWarps, 0, s>>>(r.p);
  });
  return launch_status();
}

// ------------------------------------------------------------------ clipping
constexpr int kGradTensors = 768;     // tensors of one launch (24 KB of kernel parameters)
constexpr int kGradTensorsSmall = 96; // a table that small calls pass instead (3 KB)

int check_list(const orda_tensor_list_t* l) {
  if (!l || l->abi_version != ORDA_ABI_VERSION || l->count < 0) return ORDA_ERR_INVALID_ARGUMENT;
  if (l->count > 0 && (!l->src || !l->numel || !l->dtype)) return ORDA_ERR_INVALID_ARGUMENT;
  for (int i = 0; i < l->count; ++i) {
    if (l->numel[i] < 0 || !float_dtype(l->dtype[i])) return ORDA_ERR_INVALID_ARGUMENT;
    if (l->numel[i] == 0) continue;
    if (!l->src[i] || (l->dst && !l->dst[i])) return ORDA_ERR_INVALID_ARGUMENT;
    const uintptr_t es = esize(l->dtype[i]);
    if (reinterpret_cast<uintptr_t>(l->src[i]) % es || (l->dst && reinterpret_cast<uintptr_t>(l->dst[i]) % es))
      return ORDA_ERR_ALIGNMENT;
  }
  return ORDA_OK;
}

int grad_blocks() { return 8 * num_sms(); }
int grad_launches(int count) { return static_cast<int>(cdiv(std::max(count, 1), kGradTensors)); }

// Table of tensors [first, last) of the list; returns its number of chunks, or -1 if there are too many.
// Four chunks a block, so that the blocks end together without a search for every few loads, but none
// smaller than one pass of a block's threads or larger than 64 Ki elements. (A list of 124M bf16 values is
// read in 47 us; with one or two 64 Ki-element chunks a block it took 49, with sixteen smaller ones 53.)
template <int N>
int64_t fill_table(const orda_tensor_list_t* l, int first, int last, int blocks, GradTable<N>& g) {
  int64_t total = 0;
  for (int i = first; i < last; ++i) total += l->numel[i];
  const int64_t step = 8 * kGradThreads;
  g.chunk = static_cast<int32_t>(std::min<int64_t>(std::max<int64_t>(cdiv(cdiv(total, 4 * blocks), step), 1) * step, 65536));
  g.count = last - first;
  int64_t chunks = 0;
  for (int i = first; i < last; ++i) {
    const int k = i - first;
    g.src[k] = l->src[i];
    g.dst[k] = l->dst ? l->dst[i] : nullptr;
    g.numel[k] = l->numel[i];
    g.dtype[k] = static_cast<uint8_t>(l->dtype[i]);
    g.first_chunk[k] = static_cast<int32_t>(chunks);
    chunks += cdiv(l->numel[i], g.chunk);
    if (chunks > INT32_MAX) return -1;
  }
  g.first_chunk[g.count] = static_cast<int32_t>(chunks);
  return chunks;
}

template <int N>
int clip_launches(const orda_tensor_list_t* l, double max_norm, double eps, float* norm, double* partial,
                  cudaStream_t s) {
  const int blocks = grad_blocks();
  static thread_local GradTable<N> g;
  int parts = 0;
  for (int pass = 0; pass < 2; ++pass) {
    bool norm_out = false;
    for (int first = 0; first < l->count || first == 0; first += N) {
      const int last = std::min(l->count, first + N);
      // one table serves both launches of a call that has only one
      if (pass == 0 || l->count > N)
        if (fill_table(l, first, last, blocks, g) < 0) return ORDA_ERR_UNSUPPORTED;
      const int grid = std::max(1, std::min<int>(g.first_chunk[g.count], blocks));
      count_launch();
      if (pass == 0) {
        grad_squares_kernel<N><<<grid, kGradThreads, 0, s>>>(g, partial + parts);
        parts += grid;
      } else {
        grad_scale_kernel<N><<<grid, kGradThreads, 0, s>>>(g, partial, parts, max_norm, eps, norm_out ? nullptr : norm);
        norm_out = true;
      }
      if (l->count == 0) break;
    }
    if (pass == 0 && !l->dst) {
      count_launch();
      grad_norm_kernel<<<1, kGradThreads, 0, s>>>(partial, parts, norm);
      break;
    }
  }
  return launch_status();
}

}  // namespace

extern "C" {

int32_t orda_rotary_turns(const double* radians, int32_t n, uint64_t* out) {
  if (n < 0 || (n > 0 && (!radians || !out))) return ORDA_ERR_INVALID_ARGUMENT;
  const long double two_pi = 6.283185307179586476925286766559L;
  for (int32_t i = 0; i < n; ++i) {
    if (!std::isfinite(radians[i])) return ORDA_ERR_INVALID_ARGUMENT;
    long double turn = radians[i] / two_pi;
    turn -= floorl(turn);
    turn *= 18446744073709551616.0L;
    out[i] = turn < 18446744073709551616.0L ? static_cast<uint64_t>(turn) : 0u;  // (a tiny negative angle rounds to a whole turn)
  }
  return ORDA_OK;
}

int32_t orda_rotary_forward(const orda_rotary_args_t* args, void* stream) {
  const int rc = check_rotary(args, false);
  if (rc) return rc;
  if (args->batch * args->seq == 0 || args->heads[0] + args->heads[1] == 0) return ORDA_OK;
  const RotaryPlan r = plan_rotary(args, false);
  const bool norm = args->weight[0] != nullptr;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (args->dtype) {
    case ORDA_BF16: return dispatch_rotary<__nv_bfloat16>(r, norm, s);
    case ORDA_F16: return dispatch_rotary<__half>(r, norm, s);
    default: return dispatch_rotary<float>(r, norm, s);
  }
}

size_t orda_qk_norm_rotary_backward_workspace_bytes(const orda_rotary_args_t* args) {
  if (check_rotary(args, true) != ORDA_OK) return 0;
  return align256(sizeof(float) * 2 * args->head_dim * 4 * static_cast<size_t>(num_sms()));
}

int32_t orda_qk_norm_rotary_backward(const orda_rotary_args_t* args, void* workspace, size_t workspace_bytes,
                                     void* stream) {
  int rc = check_rotary(args, true);
  if (rc) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (args->batch * args->seq == 0 || args->heads[0] + args->heads[1] == 0) {
    for (int i = 0; i < 2; ++i) cudaMemsetAsync(args->dweight[i], 0, esize(args->weight_dtype) * args->head_dim, s);
    return launch_status();
  }
  if (!workspace || workspace_bytes < orda_qk_norm_rotary_backward_workspace_bytes(args)) return ORDA_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) & 15u) return ORDA_ERR_ALIGNMENT;
  RotaryPlan r = plan_rotary(args, true);
  r.p.dw_partial = static_cast<float*>(workspace);
  switch (args->dtype) {
    case ORDA_BF16: rc = dispatch_norm_backward<__nv_bfloat16>(r, s); break;
    case ORDA_F16: rc = dispatch_norm_backward<__half>(r, s); break;
    default: rc = dispatch_norm_backward<float>(r, s); break;
  }
  if (rc) return rc;
  count_launch();
  norm_weight_grad_kernel<<<dim3(static_cast<unsigned>(cdiv(args->head_dim, kNormSumCols)), 2), 1024, 0, s>>>(
      r.p.dw_partial, r.grid, args->head_dim, args->weight_dtype, args->dweight[0], args->dweight[1]);
  return launch_status();
}

size_t orda_clip_workspace_bytes(const orda_tensor_list_t* list) {
  if (check_list(list) != ORDA_OK) return 0;
  return align256(sizeof(double) * static_cast<size_t>(grad_blocks()) * grad_launches(list->count));
}

int32_t orda_clip_gradients(const orda_tensor_list_t* list, double max_norm, double eps, float* norm, void* workspace,
                            size_t workspace_bytes, void* stream) {
  const int rc = check_list(list);
  if (rc) return rc;
  if (!norm || !(max_norm >= 0.0) || !(eps >= 0.0)) return ORDA_ERR_INVALID_ARGUMENT;
  if (!workspace || workspace_bytes < orda_clip_workspace_bytes(list)) return ORDA_ERR_WORKSPACE;
  if ((reinterpret_cast<uintptr_t>(workspace) & 15u) || (reinterpret_cast<uintptr_t>(norm) & 3u)) return ORDA_ERR_ALIGNMENT;
  double* partial = static_cast<double*>(workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (list->count <= kGradTensorsSmall) return clip_launches<kGradTensorsSmall>(list, max_norm, eps, norm, partial, s);
  return clip_launches<kGradTensors>(list, max_norm, eps, norm, partial, s);
}

}  // extern "C"
