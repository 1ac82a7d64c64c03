// Python binding of include/orda_b200_student.h (module orda_ce_kernel._student): argument checks, output
// and workspace allocation, and the autograd nodes of the student-step operators.
//
// These operators run for a few microseconds where a student decodes, so what the host does per call
// decides their speed; filling the C structs from Python through ctypes took 30 us a call for a
// rotation whose kernel runs 5. The loss, one long call per step, stays on ctypes.
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/autocast_mode.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/CUDAGraphsUtils.cuh>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/custom_class.h>

#include <algorithm>

#include "orda_b200_student.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void check_status(int32_t rc, const char* what) {
  TORCH_CHECK(rc == ORDA_OK, what, " failed: ", orda_status_string(rc), " (status ", rc, ")");
}

bool supported(at::ScalarType t) { return t == at::kFloat || t == at::kHalf || t == at::kBFloat16; }

int32_t dtype_code(at::ScalarType t) { return t == at::kFloat ? ORDA_F32 : t == at::kHalf ? ORDA_F16 : ORDA_BF16; }

// Every tensor on one CUDA device that the kernels were built for.
void require_cuda(const char* what, const Tensor& first, std::initializer_list<const Tensor*> rest) {
  for (const Tensor* t : rest)
    TORCH_CHECK_VALUE(t->device() == first.device(), what, ": tensors are on ", first.device(), " and ", t->device());
  bool ok = first.is_cuda() && first.layout() == at::kStrided;
  if (ok) {
    const cudaDeviceProp* p = at::cuda::getDeviceProperties(first.get_device());
    ok = p->major == 10 && p->minor == 0;
  }
  TORCH_CHECK(ok, what, " requires CUDA tensors on a B200 (sm_100a) GPU and the built CUDA library; "
              "there is no CPU fallback");
}

Tensor new_empty(at::IntArrayRef size, at::ScalarType dtype, const Tensor& like) {
  return Tensor(at::detail::empty_cuda(size, dtype, like.device(), std::nullopt));
}

// A tensor that a kernel reads by the sizes of another one.
void require_like(const char* what, const Tensor& t, at::IntArrayRef size, const Tensor& like) {
  TORCH_CHECK_VALUE(t.sizes() == size && t.scalar_type() == like.scalar_type() && t.device() == like.device(), what,
                    " must have shape ", size, ", ", like.scalar_type(), ", on ", like.device(), ", got ", t.sizes(), ", ",
                    t.scalar_type(), ", on ", t.device());
}

// Something records the calls that pass through PyTorch's dispatcher: these do not, and take the custom ops instead
// (an empty result tells the caller to).
bool recorded() {
  return c10::impl::TorchDispatchModeTLS::any_modes_set() ||
         c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch) || torch::jit::tracer::isTracing();
}

// For the calls that have no custom op: a graph would hold their results of this run as constants. (Modes that
// only watch, such as a FLOP counter, do no harm.)
void refuse_graph_recording(const char* what) {
  TORCH_CHECK(!c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY) &&
                  !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch) &&
                  !torch::jit::tracer::isTracing(),
              what, " cannot be recorded into a graph; call it outside of the traced function");
}

// There is no forward-mode derivative; a result without a tangent would count as a constant.
void refuse_tangent(const char* what, const Tensor& t) {
  TORCH_CHECK(!t._fw_grad(0).defined(), what, " has no forward-mode derivative, and an input carries a tangent");
}

// The tensor with its values in memory: not a view that stands for their negatives, nor a zero tensor without any.
Tensor plain(const Tensor& t) {
  if (t._is_zerotensor()) return t.clone();
  return t.is_neg() ? t.resolve_neg() : t;
}

// A tensor in the memory of `whole` that is no view of it: writes to one part do not count as writes to another.
Tensor part_of(const Tensor& whole, at::IntArrayRef size, at::IntArrayRef stride, int64_t offset, caffe2::TypeMeta dtype) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(whole.storage()),
                                                      c10::DispatchKeySet(c10::DispatchKey::CUDA), dtype);
  t.unsafeGetTensorImpl()->set_sizes_and_strides(size, stride, offset);
  return t;
}

// A zeroed device word for the kernels' bounded waits.
Tensor new_status(const Tensor& like, cudaStream_t s) {
  Tensor t = new_empty({1}, at::kInt, like);
  C10_CUDA_CHECK(cudaMemsetAsync(t.data_ptr(), 0, sizeof(int32_t), s));
  return t;
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

int64_t round8(int64_t v) { return (v + 7) / 8 * 8; }

// Gradients of a backward pass that was itself recorded (create_graph) may be read but not differentiated.
variable_list differentiable_once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list out;
  for (auto& g : grads) {
    if (!g.defined()) {
      out.push_back(g);
      continue;
    }
    g = g.detach();
    g.set_requires_grad(true);
    auto fn = std::make_shared<torch::autograd::DelayedError>(
        "trying to differentiate twice a function that was marked with @once_differentiable", 1);
    out.push_back((*fn)({g})[0]);
  }
  return out;
}

// A captured backward pass whose gradients go on to a node of the default stream - a leaf that an eager graph
// still holds, or a cast made before the capture - would have autograd make that stream wait for the
// capture, which CUDA forbids and which ends the process. Refused here, before anything is launched.
void refuse_eager_nodes_in_capture(const char* what) {
  const auto node = torch::autograd::get_current_node();
  const auto here = at::cuda::getCurrentCUDAStream();
  if (!node || here.stream() == nullptr ||
      at::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None)
    return;
  for (size_t i = 0; i < node->num_outputs(); ++i) {
    if (!node->should_compute_output(i) || !node->task_should_compute_output(i)) continue;
    const auto stream = node->next_edge(i).function->stream();
    TORCH_CHECK(!stream || c10::cuda::CUDAStream(*stream).stream() != nullptr, what,
                ": the backward pass is captured into a CUDA graph, but input ", i,
                " belongs to an autograd graph that was recorded on the default stream and still lives; drop that "
                "graph (or record it on a side stream) before the capture");
  }
}

// ------------------------------------------------------------------ gated feed-forward block
int32_t activation_code(const std::string& name) {
  if (name == "silu") return ORDA_ACT_SILU;
  if (name == "gelu") return ORDA_ACT_GELU;
  if (name == "gelu_tanh") return ORDA_ACT_GELU_TANH;
  if (name == "relu") return ORDA_ACT_RELU;
  TORCH_CHECK_VALUE(false, "activation must be one of 'gelu', 'gelu_tanh', 'relu' and 'silu', got '", name, "'");
}

// Row stride of a 2-D operand; a single row's stride means nothing, so its length stands for it.
int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

// The operands (one dtype) as the kernels read them: contiguous columns and 16-byte aligned rows, in 16 bits
// of a multiple of 8 elements. Copied only where they are not; the copies are no part of the autograd graph.
struct GluOperands {
  Tensor t[3];  // x, gate, up
  int64_t hidden;

  GluOperands(const Tensor& x, const Tensor& gate, const Tensor& up) : t{x, gate, up}, hidden(x.size(1)) {
    at::AutoGradMode off(false);
    TORCH_CHECK_VALUE(gate.scalar_type() == x.scalar_type() && up.scalar_type() == x.scalar_type(),
                      "gated_linear_unit: operands must have one dtype, got ", x.scalar_type(), ", ",
                      gate.scalar_type(), " and ", up.scalar_type());
    const bool wide = x.scalar_type() == at::kFloat;
    if (wide || hidden % 8 == 0) {
      const int64_t unit = wide ? 1 : 8;
      for (Tensor& o : t) {
        const int64_t ld = row_stride(o);
        if ((o.stride(1) != 1 && o.size(1) > 1) || ld % unit || ld < o.size(1)) o = o.contiguous();
        if (reinterpret_cast<uintptr_t>(o.data_ptr()) % 16) o = o.clone(at::MemoryFormat::Contiguous);
      }
      return;
    }
    const void* src[3];
    void* dst[3];
    int64_t ld[3], rows[3];
    Tensor padded[3];
    for (int i = 0; i < 3; ++i) {
      if (t[i].stride(1) != 1 && hidden > 1) t[i] = t[i].contiguous();
      padded[i] = new_empty({t[i].size(0), round8(hidden)}, x.scalar_type(), x);
      src[i] = t[i].data_ptr();
      dst[i] = padded[i].data_ptr();
      ld[i] = row_stride(t[i]);
      rows[i] = t[i].size(0);
    }
    c10::cuda::CUDAGuard guard(x.device());
    check_status(orda_pad_rows(3, src, ld, rows, hidden, dst, at::cuda::getCurrentCUDAStream().stream()),
                 "orda_pad_rows");
    for (int i = 0; i < 3; ++i) t[i] = padded[i];
  }
};

// Returns the number of rows.
int64_t check_glu_shapes(const Tensor& x, const Tensor& gate, const Tensor& up) {
  TORCH_CHECK_VALUE(gate.dim() == 2 && gate.sizes() == up.sizes(),
                    "gate_weight and up_weight must have one shape (ffn, hidden), got ", gate.sizes(), " and ", up.sizes());
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) == gate.size(1), "x must have shape (..., ", gate.size(1), "), got ",
                    x.sizes());
  TORCH_CHECK_VALUE(gate.numel() > 0, "gate_weight must not be empty, got shape=", gate.sizes());
  for (const Tensor* t : {&x, &gate, &up})
    TORCH_CHECK_VALUE(supported(t->scalar_type()), "gated_linear_unit: tensors must be float32, float16 or bfloat16, got ",
                      t->scalar_type());
  return x.numel() / x.size(-1);
}

void check_glu(const Tensor& x, const Tensor& gate, const Tensor& up) {
  check_glu_shapes(x, gate, up);
  require_cuda("gated_linear_unit", x, {&gate, &up});
}

orda_glu_args_t glu_args(const Tensor& x, const Tensor& gate, const Tensor& up, int64_t act) {
  orda_glu_args_t a{};
  a.abi_version = ORDA_ABI_VERSION;
  a.dtype = dtype_code(x.scalar_type());
  a.activation = static_cast<int32_t>(act);
  a.rows = x.size(0);
  a.hidden = x.size(1);
  a.ffn = gate.size(0);
  a.x = x.data_ptr();
  a.ld_x = row_stride(x);
  a.gate = gate.data_ptr();
  a.ld_gate = row_stride(gate);
  a.up = up.data_ptr();
  a.ld_up = row_stride(up);
  a.ld_h = a.ffn;
  a.ld_pre = round8(a.ffn);
  a.grad_cols = a.hidden;
  return a;
}

// h [rows, ffn] and, where `save`, the two products before the activation as [2, rows, ceil8(ffn)].
std::pair<Tensor, Tensor> glu_forward(const Tensor& x, const Tensor& gate, const Tensor& up, int64_t act, bool save) {
  c10::cuda::CUDAGuard guard(x.device());
  cudaStream_t s = at::cuda::getCurrentCUDAStream().stream();
  orda_glu_args_t a = glu_args(x, gate, up, act);
  const auto dt = x.scalar_type();
  Tensor h = new_empty({a.rows, a.ld_h}, dt, x), pre, status;
  if (save || dt == at::kFloat) {
    pre = new_empty({2, a.rows, a.ld_pre}, dt, x);
    a.pre_gate = pre.data_ptr();
    a.pre_up = static_cast<char*>(pre.data_ptr()) + a.rows * a.ld_pre * pre.element_size();
  }
  if (a.rows > ORDA_GLU_FEW_ROWS && dt != at::kFloat) status = new_status(x, s);
  a.h = h.data_ptr();
  a.device_status = static_cast<int32_t*>(ptr(status));
  check_status(orda_glu_forward(&a, s), "orda_glu_forward");
  return {h, pre};
}

// (dx, gradients of both weights), `hidden` columns each: the latter [ceil8(ffn) + ffn, hidden], gate's from
// row 0, up's from row ceil8(ffn).
std::pair<Tensor, Tensor> glu_backward(Tensor dh, const Tensor& x, const Tensor& gate, const Tensor& up,
                                       Tensor pre, int64_t act, int64_t hidden, bool need_x, bool need_w) {
  c10::cuda::CUDAGuard guard(x.device());
  cudaStream_t s = at::cuda::getCurrentCUDAStream().stream();
  orda_glu_args_t a = glu_args(x, gate, up, act);
  const auto dt = x.scalar_type();
  Tensor dx, dw, ws, status;
  a.grad_cols = hidden;
  if (need_x) dx = new_empty({a.rows, hidden}, dt, x);
  if (need_w) dw = new_empty({a.ld_pre + a.ffn, hidden}, dt, x);
  if (a.rows == 0) {
    if (dw.defined()) dw.zero_();
    return {dx, dw};
  }
  dh = plain(dh).contiguous();
  pre = plain(pre).contiguous();
  if (reinterpret_cast<uintptr_t>(pre.data_ptr()) % 16) pre = pre.clone();
  a.pre_gate = pre.data_ptr();
  a.pre_up = static_cast<char*>(pre.data_ptr()) + a.rows * a.ld_pre * pre.element_size();
  a.dh = dh.data_ptr();
  a.dx = ptr(dx);
  a.dweights = ptr(dw);
  if (dt != at::kFloat) status = new_empty({1}, at::kInt, x);  // the call clears it
  a.device_status = static_cast<int32_t*>(ptr(status));
  const size_t bytes = orda_glu_backward_workspace_bytes(&a);
  ws = new_empty({static_cast<int64_t>(bytes)}, at::kByte, x);
  check_status(orda_glu_backward(&a, ws.data_ptr(), bytes, s), "orda_glu_backward");
  return {dx, dw};
}

struct GluFunction : torch::autograd::Function<GluFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& gate, const Tensor& up, int64_t act) {
    const GluOperands o(x, gate, up);
    auto [h, pre] = glu_forward(o.t[0], o.t[1], o.t[2], act, true);
    ctx->save_for_backward({o.t[0], o.t[1], o.t[2], pre});
    ctx->saved_data["act"] = act;
    ctx->saved_data["hidden"] = o.hidden;
    return h;
  }
  static variable_list backward(AutogradContext* ctx, variable_list dh) {
    refuse_eager_nodes_in_capture("gated_linear_unit");
    const auto saved = ctx->get_saved_variables();
    const bool need_x = ctx->needs_input_grad(0), need_g = ctx->needs_input_grad(1), need_u = ctx->needs_input_grad(2);
    variable_list grads(4);
    {
      at::AutoGradMode off(false);
      // what a saved-tensor hook returns may lie in memory in another way, and must be looked at again
      check_glu(saved[0], saved[1], saved[2]);
      const GluOperands o(plain(saved[0]), plain(saved[1]), plain(saved[2]));
      const int64_t ffn = saved[1].size(0), pre_size[3] = {2, saved[0].size(0), round8(ffn)};
      require_like("gated_linear_unit: the products of the forward pass", saved[3], pre_size, saved[0]);
      const int64_t dh_size[2] = {saved[0].size(0), ffn};
      require_like("gated_linear_unit: the gradient", dh[0], dh_size, saved[0]);
      auto [dx, dw] = glu_backward(dh[0], o.t[0], o.t[1], o.t[2], saved[3], ctx->saved_data["act"].toInt(),
                                   ctx->saved_data["hidden"].toInt(), need_x, need_g || need_u);
      grads[0] = dx;
      const int64_t size[2] = {ffn, ctx->saved_data["hidden"].toInt()}, stride[2] = {size[1], 1};
      if (need_g) grads[1] = part_of(dw, size, stride, 0, dw.dtype());
      if (need_u) grads[2] = part_of(dw, size, stride, round8(ffn) * size[1], dw.dtype());
    }
    return differentiable_once(std::move(grads));
  }
};

// The loss's rule: an active autocast dtype wins, else bf16 if any input is bf16, else fp16, else fp32.
at::ScalarType compute_dtype(std::initializer_list<const Tensor*> tensors) {
  if (at::autocast::is_autocast_enabled(at::kCUDA)) {
    const auto t = at::autocast::get_autocast_dtype(at::kCUDA);
    if (t == at::kBFloat16 || t == at::kHalf) return t;
  }
  for (auto dt : {at::kBFloat16, at::kHalf})
    for (const Tensor* t : tensors)
      if (t->scalar_type() == dt) return dt;
  return at::kFloat;
}

std::optional<Tensor> gated_linear_unit(const Tensor& x, const Tensor& gate_weight, const Tensor& up_weight,
                                        const std::string& activation) {
  const int64_t act = activation_code(activation);
  for (const Tensor* t : {&x, &gate_weight, &up_weight}) refuse_tangent("gated_linear_unit", *t);
  if (recorded()) return std::nullopt;
  check_glu(x, gate_weight, up_weight);
  const auto dt = compute_dtype({&gate_weight, &up_weight, &x});
  auto cast = [dt](const Tensor& t) { return plain(t.scalar_type() == dt ? t : t.to(dt)); };
  const Tensor flat = cast(x.dim() == 2 ? x : x.reshape({-1, x.size(-1)})), gate = cast(gate_weight), up = cast(up_weight);
  Tensor h;
  if (at::GradMode::is_enabled() && (flat.requires_grad() || gate.requires_grad() || up.requires_grad())) {
    h = GluFunction::apply(flat, gate, up, act);
  } else {
    const GluOperands o(flat, gate, up);
    h = glu_forward(o.t[0], o.t[1], o.t[2], act, false).first;
  }
  if (x.dim() == 2) return h;
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end() - 1);
  shape.push_back(gate.size(0));
  return h.view(shape);
}

// Without autograd, for the custom ops: x any number of dimensions, all tensors in the compute dtype.
std::tuple<Tensor, Tensor> glu_forward_op(const Tensor& x, const Tensor& gate, const Tensor& up, int64_t act) {
  check_glu(x, gate, up);
  const GluOperands o(plain(x.reshape({-1, x.size(-1)})), plain(gate), plain(up));
  auto [h, pre] = glu_forward(o.t[0], o.t[1], o.t[2], act, true);
  // an op's outputs are compared and kept whole: no memory behind the last feature that holds anything
  const int64_t ffn = gate.size(0);
  if (pre.size(2) > ffn) pre.slice(2, ffn).zero_();
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end() - 1);
  shape.push_back(gate.size(0));
  return {h.view(shape), pre};
}

std::tuple<Tensor, Tensor, Tensor> glu_backward_op(const Tensor& dh, const Tensor& x, const Tensor& gate,
                                                   const Tensor& up, const Tensor& pre, int64_t act) {
  const int64_t rows = check_glu_shapes(x, gate, up), ffn = gate.size(0), hidden = x.size(-1);
  const int64_t pre_size[3] = {2, rows, round8(ffn)};
  require_like("gated_linear_unit: the products of the forward pass", pre, pre_size, x);
  std::vector<int64_t> dh_size(x.sizes().begin(), x.sizes().end() - 1);
  dh_size.push_back(ffn);
  require_like("gated_linear_unit: the gradient", dh, dh_size, x);
  require_cuda("gated_linear_unit", x, {&gate, &up});
  const GluOperands o(plain(x.reshape({-1, hidden})), plain(gate), plain(up));
  auto [dx, dw] = glu_backward(dh.reshape({-1, ffn}), o.t[0], o.t[1], o.t[2], pre, act, hidden, true, true);
  // an op's outputs share no storage
  return {dx.view(x.sizes()), dw.slice(0, 0, ffn).clone(), dw.slice(0, round8(ffn)).clone()};
}

// ------------------------------------------------------------------ rotary positions
// What a RotaryConfig says, in the form the kernels take.
struct RotaryPlan : torch::CustomClassHolder {
  std::vector<uint64_t> turns;
  int32_t head_dim, rotary_dim, layout;
  float magnitude;
  RotaryPlan(const std::vector<double>& frequencies, int64_t head_dim_, bool interleaved, double magnitude_)
      : turns(frequencies.size()), head_dim(static_cast<int32_t>(head_dim_)),
        rotary_dim(static_cast<int32_t>(2 * frequencies.size())),
        layout(interleaved ? ORDA_ROTARY_INTERLEAVED : ORDA_ROTARY_HALF), magnitude(static_cast<float>(magnitude_)) {
    TORCH_CHECK_VALUE(head_dim >= rotary_dim && head_dim <= ORDA_ROTARY_MAX_DIM, "rotary plan of ", rotary_dim, " of ",
                      head_dim, " elements");
    check_status(orda_rotary_turns(frequencies.data(), static_cast<int32_t>(turns.size()), turns.data()),
                 "orda_rotary_turns");
  }
};
using PlanPtr = c10::intrusive_ptr<RotaryPlan>;

void check_qk(const char* what, const Tensor& q, const Tensor& k, const Tensor& positions, const RotaryPlan& plan) {
  TORCH_CHECK_VALUE((q.dim() == 3 || q.dim() == 4) && k.dim() == q.dim() &&
                        q.sizes().slice(0, q.dim() - 2) == k.sizes().slice(0, q.dim() - 2),
                    what, ": q and k must be (batch, seq, heads, head_dim) or (tokens, heads, head_dim) with the same "
                    "tokens, got ", q.sizes(), " and ", k.sizes());
  TORCH_CHECK_VALUE(q.size(-1) == plan.head_dim && k.size(-1) == plan.head_dim, what,
                    ": heads must have config.head_dim=", plan.head_dim, " elements, got ", q.size(-1), " and ", k.size(-1));
  TORCH_CHECK_VALUE(std::max(q.size(-2), k.size(-2)) <= ORDA_ROTARY_MAX_HEADS, what, ": at most ", ORDA_ROTARY_MAX_HEADS,
                    " heads each, got ", q.size(-2), " and ", k.size(-2));
  TORCH_CHECK_VALUE(supported(q.scalar_type()) && k.scalar_type() == q.scalar_type(), what,
                    ": q and k must both be float32, float16 or bfloat16, got ", q.scalar_type(), " and ",
                    k.scalar_type());
  TORCH_CHECK_VALUE(positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong, what,
                    ": positions must be int32 or int64, got ", positions.scalar_type());
  const auto tokens = q.sizes().slice(0, q.dim() - 2);
  TORCH_CHECK_VALUE(positions.sizes() == tokens || positions.sizes() == tokens.slice(tokens.size() - 1), what,
                    ": positions must have shape ", tokens, " or ", tokens.slice(tokens.size() - 1), ", got ",
                    positions.sizes());
}

void check_norm_weights(const char* what, const Tensor& wq, const Tensor& wk, const RotaryPlan& plan, double eps) {
  TORCH_CHECK_VALUE(wq.dim() == 1 && wq.size(0) == plan.head_dim, what, ": q_weight must have shape (", plan.head_dim,
                    ",), got ", wq.sizes());
  TORCH_CHECK_VALUE(wk.dim() == 1 && wk.size(0) == plan.head_dim, what, ": k_weight must have shape (", plan.head_dim,
                    ",), got ", wk.sizes());
  TORCH_CHECK_VALUE(supported(wq.scalar_type()) && wk.scalar_type() == wq.scalar_type(), what,
                    ": weights must have one dtype of float32, float16 and bfloat16, got ", wq.scalar_type(), " and ",
                    wk.scalar_type());
  TORCH_CHECK_VALUE(eps >= 0.0, what, ": eps must be >= 0, got ", eps);
}

Tensor dense_last(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? plain(t) : plain(t.contiguous()); }

// Element strides of batch, sequence and heads; the stride of a dimension of one means nothing and counts as 0.
void strides_of(const Tensor& t, int64_t (&out)[3]) {
  const int o = t.dim() == 4;
  auto stride = [&](int d) { return t.size(d) > 1 ? t.stride(d) : 0; };
  out[0] = o ? stride(0) : 0;
  out[1] = stride(o);
  out[2] = stride(o + 1);
}

orda_rotary_args_t rotary_args(const Tensor& q, const Tensor& k, const Tensor& positions, const RotaryPlan& plan,
                               const Tensor& out_q, const Tensor& out_k) {
  orda_rotary_args_t a{};
  a.abi_version = ORDA_ABI_VERSION;
  a.dtype = dtype_code(q.scalar_type());
  const bool batched = q.dim() == 4;
  a.batch = batched ? q.size(0) : 1;
  a.seq = q.size(batched);
  a.heads[0] = static_cast<int32_t>(q.size(-2));
  a.heads[1] = static_cast<int32_t>(k.size(-2));
  a.head_dim = plan.head_dim;
  a.rotary_dim = plan.rotary_dim;
  a.layout = plan.layout;
  a.x[0] = q.data_ptr();
  a.x[1] = k.data_ptr();
  strides_of(q, a.x_stride[0]);
  strides_of(k, a.x_stride[1]);
  a.out[0] = out_q.data_ptr();
  a.out[1] = out_k.data_ptr();
  strides_of(out_q, a.out_stride[0]);
  strides_of(out_k, a.out_stride[1]);
  a.positions = positions.data_ptr();
  a.position_stride[0] = positions.dim() == 2 ? positions.stride(0) : 0;
  a.position_stride[1] = positions.stride(-1);
  a.positions_int64 = positions.scalar_type() == at::kLong;
  a.turns = plan.turns.data();
  a.magnitude = plan.magnitude;
  return a;
}

void set_weights(orda_rotary_args_t& a, const Tensor& wq, const Tensor& wk, double eps) {
  a.weight_dtype = dtype_code(wq.scalar_type());
  a.weight[0] = wq.data_ptr();
  a.weight[1] = wk.data_ptr();
  a.eps = static_cast<float>(eps);
}

variable_list rotate(const Tensor& q, const Tensor& k, const Tensor& positions, const RotaryPlan& plan, bool inverse,
                     const Tensor& wq, const Tensor& wk, double eps) {
  c10::cuda::CUDAGuard guard(q.device());
  Tensor out_q = new_empty(q.sizes(), q.scalar_type(), q), out_k = new_empty(k.sizes(), k.scalar_type(), k);
  orda_rotary_args_t a = rotary_args(q, k, positions, plan, out_q, out_k);
  a.inverse = inverse;
  if (wq.defined()) set_weights(a, wq, wk, eps);
  check_status(orda_rotary_forward(&a, at::cuda::getCurrentCUDAStream().stream()), "orda_rotary_forward");
  return {out_q, out_k};
}

// Gradients of q, k and the two weights.
variable_list norm_rotate_backward(const Tensor& dq, const Tensor& dk, const Tensor& q, const Tensor& k,
                                   const Tensor& wq, const Tensor& wk, const Tensor& positions, const RotaryPlan& plan,
                                   double eps) {
  c10::cuda::CUDAGuard guard(q.device());
  const Tensor dy[2] = {dense_last(dq), dense_last(dk)};
  Tensor gq = new_empty(q.sizes(), q.scalar_type(), q), gk = new_empty(k.sizes(), k.scalar_type(), k);
  Tensor gwq = new_empty(wq.sizes(), wq.scalar_type(), q), gwk = new_empty(wk.sizes(), wk.scalar_type(), q);
  orda_rotary_args_t a = rotary_args(q, k, positions, plan, gq, gk);
  set_weights(a, wq, wk, eps);
  for (int i = 0; i < 2; ++i) {
    a.dy[i] = dy[i].data_ptr();
    strides_of(dy[i], a.dy_stride[i]);
  }
  a.dweight[0] = gwq.data_ptr();
  a.dweight[1] = gwk.data_ptr();
  const size_t bytes = orda_qk_norm_rotary_backward_workspace_bytes(&a);
  const Tensor ws = new_empty({static_cast<int64_t>(bytes)}, at::kByte, q);
  check_status(orda_qk_norm_rotary_backward(&a, ws.data_ptr(), bytes, at::cuda::getCurrentCUDAStream().stream()),
               "orda_qk_norm_rotary_backward");
  return {gq, gk, gwq, gwk};
}

// The same of tensors that come from outside: a custom op's arguments, or what a saved-tensor hook returned.
variable_list checked_norm_rotate_backward(const Tensor& dq, const Tensor& dk, const Tensor& q, const Tensor& k,
                                           const Tensor& wq, const Tensor& wk, const Tensor& positions,
                                           const RotaryPlan& plan, double eps) {
  check_qk("qk_norm_rotary", q, k, positions, plan);
  check_norm_weights("qk_norm_rotary", wq, wk, plan, eps);
  require_like("qk_norm_rotary: the gradient of the queries", dq, q.sizes(), q);
  require_like("qk_norm_rotary: the gradient of the keys", dk, k.sizes(), k);
  require_cuda("qk_norm_rotary", q, {&k, &positions, &wq, &wk});
  return norm_rotate_backward(dq, dk, dense_last(q), dense_last(k), plain(wq).contiguous(),
                              plain(wk).contiguous(), plain(positions), plan, eps);
}

struct RotaryFunction : torch::autograd::Function<RotaryFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& positions,
                               PlanPtr plan) {
    ctx->save_for_backward({positions});
    ctx->saved_data["plan"] = c10::IValue::make_capsule(plan);
    return rotate(q, k, positions, *plan, false, {}, {}, 0.0);
  }
  static variable_list backward(AutogradContext* ctx, variable_list dy) {
    refuse_eager_nodes_in_capture("rotary_embedding");
    const auto saved = ctx->get_saved_variables();
    const auto plan = c10::static_intrusive_pointer_cast<RotaryPlan>(ctx->saved_data["plan"].toCapsule());
    variable_list g;
    {
      at::AutoGradMode off(false);
      check_qk("rotary_embedding", dy[0], dy[1], saved[0], *plan);
      require_cuda("rotary_embedding", dy[0], {&dy[1], &saved[0]});
      g = rotate(dense_last(dy[0]), dense_last(dy[1]), plain(saved[0]), *plan, true, {}, {}, 0.0);
    }
    g.resize(4);
    return differentiable_once(std::move(g));
  }
};

struct QkNormRotaryFunction : torch::autograd::Function<QkNormRotaryFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& wq,
                               const Tensor& wk, const Tensor& positions, PlanPtr plan, double eps) {
    ctx->save_for_backward({q, k, wq, wk, positions});
    ctx->saved_data["plan"] = c10::IValue::make_capsule(plan);
    ctx->saved_data["eps"] = eps;
    return rotate(q, k, positions, *plan, false, wq, wk, eps);
  }
  static variable_list backward(AutogradContext* ctx, variable_list dy) {
    refuse_eager_nodes_in_capture("qk_norm_rotary");
    const auto s = ctx->get_saved_variables();
    const auto plan = c10::static_intrusive_pointer_cast<RotaryPlan>(ctx->saved_data["plan"].toCapsule());
    variable_list g;
    {
      at::AutoGradMode off(false);
      g = checked_norm_rotate_backward(dy[0], dy[1], s[0], s[1], s[2], s[3], s[4], *plan,
                                       ctx->saved_data["eps"].toDouble());
    }
    g.resize(7);
    return differentiable_once(std::move(g));
  }
};

std::tuple<Tensor, Tensor> two(const variable_list& v) { return {v[0], v[1]}; }

std::optional<std::tuple<Tensor, Tensor>> rotary_embedding(const Tensor& q_, const Tensor& k_, const Tensor& positions_,
                                                           PlanPtr plan) {
  check_qk("rotary_embedding", q_, k_, positions_, *plan);
  for (const Tensor* t : {&q_, &k_}) refuse_tangent("rotary_embedding", *t);
  if (recorded()) return std::nullopt;
  require_cuda("rotary_embedding", q_, {&k_, &positions_});
  const Tensor q = dense_last(q_), k = dense_last(k_), positions = plain(positions_);
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad()))
    return two(RotaryFunction::apply(q, k, positions, plan));
  return two(rotate(q, k, positions, *plan, false, {}, {}, 0.0));
}

std::optional<std::tuple<Tensor, Tensor>> qk_norm_rotary(const Tensor& q_, const Tensor& k_, const Tensor& q_weight,
                                                         const Tensor& k_weight, const Tensor& positions_, PlanPtr plan,
                                                         double eps) {
  check_qk("qk_norm_rotary", q_, k_, positions_, *plan);
  check_norm_weights("qk_norm_rotary", q_weight, k_weight, *plan, eps);
  for (const Tensor* t : {&q_, &k_, &q_weight, &k_weight}) refuse_tangent("qk_norm_rotary", *t);
  if (recorded()) return std::nullopt;
  require_cuda("qk_norm_rotary", q_, {&k_, &positions_, &q_weight, &k_weight});
  const Tensor q = dense_last(q_), k = dense_last(k_), positions = plain(positions_), wq = plain(q_weight).contiguous(),
               wk = plain(k_weight).contiguous();
  if (at::GradMode::is_enabled() &&
      (q.requires_grad() || k.requires_grad() || wq.requires_grad() || wk.requires_grad()))
    return two(QkNormRotaryFunction::apply(q, k, wq, wk, positions, plan, eps));
  return two(rotate(q, k, positions, *plan, false, wq, wk, eps));
}

// Without autograd, for the custom ops.
std::tuple<Tensor, Tensor> rotary_op(const Tensor& q, const Tensor& k, const Tensor& positions,
                                     const std::optional<Tensor>& wq, const std::optional<Tensor>& wk, double eps,
                                     bool inverse, PlanPtr plan) {
  check_qk("rotary_embedding", q, k, positions, *plan);
  TORCH_CHECK_VALUE(wq.has_value() == wk.has_value(), "qk_norm_rotary: q_weight and k_weight belong together");
  if (wq) check_norm_weights("qk_norm_rotary", *wq, *wk, *plan, eps);
  require_cuda("rotary_embedding", q, {&k, &positions});
  Tensor w[2];
  if (wq) {
    require_cuda("qk_norm_rotary", q, {&*wq, &*wk});
    w[0] = plain(*wq).contiguous();
    w[1] = plain(*wk).contiguous();
  }
  auto r = rotate(dense_last(q), dense_last(k), plain(positions), *plan, inverse, w[0], w[1], eps);
  return {r[0], r[1]};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> qk_norm_rotary_backward_op(const Tensor& dq, const Tensor& dk,
                                                                      const Tensor& q, const Tensor& k,
                                                                      const Tensor& positions, const Tensor& wq,
                                                                      const Tensor& wk, double eps, PlanPtr plan) {
  const auto r = checked_norm_rotate_backward(dq, dk, q, k, wq, wk, positions, *plan, eps);
  return {r[0], r[1], r[2], r[3]};
}

// ------------------------------------------------------------------ gradient norm and clipping
void check_limits(const char* what, double max_norm, double eps) {
  TORCH_CHECK_VALUE(max_norm >= 0.0, what, ": max_norm must be >= 0, got ", max_norm);
  TORCH_CHECK_VALUE(eps >= 0.0, what, ": eps must be >= 0, got ", eps);
}

// Tensors that are scaled in place must not share memory: a value would be scaled twice, or by two blocks at
// once. Ones with gaps between their values may lie in each other's gaps; they are scaled as copies, all made
// before anything is written.
void refuse_shared_memory(const char* what, const std::vector<Tensor>& grads) {
  struct Span {
    const char *first, *end;
    bool dense;
  };
  std::vector<Span> spans;
  spans.reserve(grads.size());
  for (const Tensor& g : grads) {
    if (g.numel() == 0) continue;
    TORCH_CHECK_VALUE(at::has_internal_overlap(g) != at::MemOverlap::Yes, what, ": a gradient of shape ", g.sizes(),
                      " holds broadcast values, which cannot be scaled in place");
    const char* first = static_cast<const char*>(g.data_ptr());
    spans.push_back({first, first + g.nbytes(), g.is_non_overlapping_and_dense()});
  }
  std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.first < b.first; });
  const char *last = nullptr, *dense_end = nullptr;
  for (const Span& s : spans) {
    TORCH_CHECK_VALUE(s.first != last, what, ": a gradient appears twice among the parameters");
    last = s.first;
    if (!s.dense) continue;
    TORCH_CHECK_VALUE(s.first >= dense_end, what, ": two gradients share memory");
    dense_end = s.end;
  }
}

void check_gradients(const char* what, const std::vector<Tensor>& grads, bool in_place = false) {
  refuse_graph_recording(what);
  for (const Tensor& g : grads) {
    refuse_tangent(what, g);
    TORCH_CHECK_VALUE(supported(g.scalar_type()), what, ": gradients must be float32, float16 or bfloat16, got ",
                      g.scalar_type());
    TORCH_CHECK_VALUE(g.layout() == at::kStrided, what, ": gradients must be strided tensors, got ", g.layout());
    TORCH_CHECK_VALUE(g.device() == grads[0].device(), what, ": tensors are on ", grads[0].device(), " and ", g.device());
  }
  if (in_place) refuse_shared_memory(what, grads);
  if (!grads.empty()) require_cuda(what, grads[0], {});
}

// A tensor whose values fill one gapless stretch of memory: itself, or a contiguous copy.
Tensor dense(const Tensor& t) { return plain(t.is_non_overlapping_and_dense() ? t : t.contiguous()); }

// Norm of `src` (0-dim fp32); `dst` (may be null) receives the clipped values. All dense, one device.
Tensor clip_call(const std::vector<Tensor>& src, const std::vector<Tensor>* dst, double max_norm, double eps) {
  c10::cuda::CUDAGuard guard(src[0].device());
  const size_t n = src.size();
  std::vector<const void*> from(n);
  std::vector<void*> to(dst ? n : 0);
  std::vector<int64_t> numel(n);
  std::vector<int32_t> code(n);
  for (size_t i = 0; i < n; ++i) {
    from[i] = src[i].data_ptr();
    if (dst) to[i] = (*dst)[i].data_ptr();
    numel[i] = src[i].numel();
    code[i] = dtype_code(src[i].scalar_type());
  }
  orda_tensor_list_t l{ORDA_ABI_VERSION, static_cast<int32_t>(n), from.data(), dst ? to.data() : nullptr, numel.data(),
                       code.data()};
  const size_t bytes = orda_clip_workspace_bytes(&l);
  Tensor norm = new_empty({}, at::kFloat, src[0]);
  const Tensor ws = new_empty({static_cast<int64_t>(bytes)}, at::kByte, src[0]);
  check_status(orda_clip_gradients(&l, max_norm, eps, norm.data_ptr<float>(), ws.data_ptr(), bytes,
                                   at::cuda::getCurrentCUDAStream().stream()),
               "orda_clip_gradients");
  return norm;
}

Tensor grad_norm(const std::vector<Tensor>& grads) {
  at::AutoGradMode off(false);
  check_gradients("grad_norm", grads);
  if (grads.empty()) return at::zeros({}, at::kFloat);
  std::vector<Tensor> src;
  src.reserve(grads.size());
  for (const Tensor& g : grads) src.push_back(dense(g));
  return clip_call(src, nullptr, 0.0, 0.0);
}

std::tuple<std::vector<Tensor>, Tensor> clip_gradients(const std::vector<Tensor>& grads, double max_norm, double eps) {
  at::AutoGradMode off(false);
  check_limits("clip_gradients", max_norm, eps);
  check_gradients("clip_gradients", grads);
  if (grads.empty()) return std::make_tuple(std::vector<Tensor>(), at::zeros({}, at::kFloat));
  std::vector<Tensor> src, out;
  src.reserve(grads.size());
  out.reserve(grads.size());
  c10::cuda::CUDAGuard guard(grads[0].device());
  int64_t bytes = 0;
  for (const Tensor& g : grads) {
    src.push_back(dense(g));
    bytes += (src.back().nbytes() + 255) / 256 * 256;
  }
  // Short lists: the host's allocations would take longer than the kernels, so the results share one.
  // (16 fp32 tensors of a 0.5M-parameter model: 25 us a call with an allocation each.)
  if (bytes <= (int64_t(16) << 20)) {
    const Tensor all = new_empty({bytes}, at::kByte, grads[0]);
    int64_t at = 0;
    for (const Tensor& d : src) {
      out.push_back(part_of(all, d.sizes(), d.strides(), at / d.element_size(), d.dtype()));
      at += (d.nbytes() + 255) / 256 * 256;
    }
  } else {
    for (const Tensor& d : src)
      out.push_back(Tensor(at::detail::empty_strided_cuda(d.sizes(), d.strides(), d.scalar_type(), d.device())));
  }
  Tensor norm = clip_call(src, &out, max_norm, eps);
  return {std::move(out), std::move(norm)};
}

Tensor clip_in_place(const std::vector<Tensor>& grads, double max_norm, double eps) {
  at::AutoGradMode off(false);
  const char* what = "clip_grad_norm_";
  check_limits(what, max_norm, eps);
  check_gradients(what, grads, true);
  if (grads.empty()) return at::zeros({}, at::kFloat);
  std::vector<Tensor> src;
  src.reserve(grads.size());
  for (const Tensor& g : grads) src.push_back(dense(g));
  Tensor norm = clip_call(src, &src, max_norm, eps);
  for (size_t i = 0; i < src.size(); ++i) {
    if (!src[i].is_same(grads[i])) grads[i].copy_(src[i]);
    else if (!grads[i].is_inference()) grads[i].unsafeGetTensorImpl()->bump_version();  // autograd sees the write
  }
  return norm;
}

}  // namespace

PYBIND11_MODULE(_student, m) {
  using torch::wrap_pybind_function_no_gil;
  py::class_<RotaryPlan, PlanPtr>(m, "RotaryPlan")
      .def(py::init<const std::vector<double>&, int64_t, bool, double>());
  m.def("refuse_eager_nodes_in_capture", wrap_pybind_function_no_gil(refuse_eager_nodes_in_capture));
  m.def("gated_linear_unit", wrap_pybind_function_no_gil(gated_linear_unit));
  m.def("glu_forward", wrap_pybind_function_no_gil(glu_forward_op));
  m.def("glu_backward", wrap_pybind_function_no_gil(glu_backward_op));
  m.def("rotary_embedding", wrap_pybind_function_no_gil(rotary_embedding));
  m.def("qk_norm_rotary", wrap_pybind_function_no_gil(qk_norm_rotary));
  m.def("rotary", wrap_pybind_function_no_gil(rotary_op));
  m.def("qk_norm_rotary_backward", wrap_pybind_function_no_gil(qk_norm_rotary_backward_op));
  m.def("grad_norm", wrap_pybind_function_no_gil(grad_norm));
  m.def("clip_gradients", wrap_pybind_function_no_gil(clip_gradients));
  m.def("clip_in_place", wrap_pybind_function_no_gil(clip_in_place));
}
