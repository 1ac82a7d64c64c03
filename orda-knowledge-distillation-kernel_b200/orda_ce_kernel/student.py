"""Operators of a student's training step around :func:`orda_ce_kernel.distillation_loss`, and of its
token-by-token run (``include/orda_b200_student.h``; the reference leaves them to PyTorch, as the model
and training loop of ``test/benchmark/src/core.py:106-138`` and ``_train.py:102-452`` do):

* :func:`gated_linear_unit` - the gated feed-forward block ``act(x Wg^T) * (x Wu^T)`` in one kernel;
* :func:`rotary_embedding` - positions rotated into queries and keys in one pass;
* :func:`qk_norm_rotary` - per-head RMS norms of queries and keys, rotated in the same pass;
* :func:`grad_norm`, :func:`clip_gradients`, :func:`clip_grad_norm_` - the global gradient norm and clipping.

The first three back-propagate (once; no double backward) and trace into one custom op each under
``torch.compile``. As for the loss there is no CPU fallback: CUDA tensors on a B200 are required. Every call
runs on the current stream of its tensors' device, takes its workspace from the caching allocator and
does not synchronise, so it can be captured into a CUDA graph.
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from functools import lru_cache
from typing import Iterable, Literal, Optional, Sequence

import torch
from torch.autograd.function import once_differentiable

from . import _native
from ._runtime import cuda_kernels_available, default_compute_dtype

Activation = Literal["silu", "gelu", "gelu_tanh", "relu"]
Layout = Literal["half", "interleaved"]
Scaling = Literal["none", "linear", "ntk", "yarn"]

_DTYPE_CODE = {torch.float32: _native.F32, torch.float16: _native.F16, torch.bfloat16: _native.BF16}
_ACT_CODE = {"silu": _native.ACT_SILU, "gelu": _native.ACT_GELU, "gelu_tanh": _native.ACT_GELU_TANH,
             "relu": _native.ACT_RELU}
_LAYOUT_CODE = {"half": _native.ROTARY_HALF, "interleaved": _native.ROTARY_INTERLEAVED}


_usable: set = set()  # devices on which the kernels were found to run


# ------------------------------------------------------------------------------------------ shared
def _require_cuda(what: str, *tensors: torch.Tensor) -> None:
    dev = tensors[0].device
    for t in tensors[1:]:
        if t.device != dev:
            raise ValueError(f"{what}: tensors are on {dev} and {t.device}")
    if dev.type == "cuda":
        if dev.index in _usable or torch.compiler.is_compiling():
            return
        if cuda_kernels_available():
            _usable.add(dev.index)
            return
    raise RuntimeError(f"{what} requires CUDA tensors on a B200 (sm_100a) GPU and the built CUDA library; "
                       "there is no CPU fallback")


class _On:
    """The tensors' device as the current one for the launches inside (free where it already is)."""

    __slots__ = ("index", "guard")

    def __init__(self, dev: torch.device):
        self.index = dev.index

    def __enter__(self):
        self.guard = None if torch.cuda.current_device() == self.index else torch.cuda.device(self.index)
        if self.guard is not None:
            self.guard.__enter__()
        return torch.cuda.current_stream(self.index).cuda_stream

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _round8(v: int) -> int:
    return (v + 7) // 8 * 8


# ------------------------------------------------------------------------------------------ gated feed-forward block
def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _ld(t: torch.Tensor) -> int:
    """Row stride of a 2-D operand; a single row's stride means nothing, so its length stands for it."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _glu_args(x, gate, up, h, pre_gate, pre_up, dh, dx, dweights, act, status):
    ffn = gate.shape[0]
    return _native.GluArgs(_native.ABI_VERSION, _DTYPE_CODE[x.dtype], act, 0, x.shape[0], x.shape[1], ffn,
                           x.data_ptr(), _ld(x), gate.data_ptr(), _ld(gate), up.data_ptr(), _ld(up),
                           _ptr(h), _round8(ffn), _ptr(pre_gate), _ptr(pre_up), _ptr(dh), _ptr(dx), _ptr(dweights),
                           status.data_ptr())


def _glu_forward(x, gate, up, act: int, save: bool):
    """h, and the products before the activation where ``save``: buffers of [rows, ceil8(ffn)]."""
    n, ffn = x.shape[0], gate.shape[0]
    fp = _round8(ffn)
    h = x.new_empty((n, fp))
    pre_gate = pre_up = None
    if save or x.dtype == torch.float32:
        pre_gate, pre_up = x.new_empty((n, fp)), x.new_empty((n, fp))
    if n:
        with _On(x.device) as stream:
            status = torch.zeros(1, dtype=torch.int32, device=x.device)
            a = _glu_args(x, gate, up, h, pre_gate, pre_up, None, None, None, act, status)
            _native.check(_native.load().orda_glu_forward(a, stream), "orda_glu_forward")
    return h, pre_gate, pre_up


def _glu_backward(dh, x, gate, up, pre_gate, pre_up, act: int, need_x: bool, need_w: bool):
    """(dx, dweights): dweights holds the gate's gradient in rows [0, ffn), up's from row ceil8(ffn)."""
    (n, hidden), ffn = x.shape, gate.shape[0]
    fp = _round8(ffn)
    dx = x.new_empty((n, hidden)) if need_x else None
    dw = x.new_empty((fp + ffn, hidden)) if need_w else None
    if n == 0:
        return dx, (dw.zero_() if dw is not None else None)
    if fp != ffn:
        dh = torch.nn.functional.pad(dh, (0, fp - ffn))
    dh = _aligned(dh if dh.is_contiguous() else dh.contiguous())
    lib = _native.load()
    with _On(x.device) as stream:
        status = torch.zeros(1, dtype=torch.int32, device=x.device)
        a = _glu_args(x, gate, up, None, pre_gate, pre_up, dh, dx, dw, act, status)
        size = int(lib.orda_glu_backward_workspace_bytes(a))
        ws = torch.empty(max(size, 16), dtype=torch.uint8, device=x.device)
        _native.check(lib.orda_glu_backward(a, ws.data_ptr(), size, stream), "orda_glu_backward")
    return dx, dw


def _aligned(t: torch.Tensor) -> torch.Tensor:
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _cast_padded(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """A 2-D operand in the compute dtype, in 16 bits with columns padded to a multiple of 8."""
    if t.dtype != dtype:
        t = t.to(dtype)
    if dtype != torch.float32 and t.shape[1] % 8:
        t = torch.nn.functional.pad(t, (0, _round8(t.shape[1]) - t.shape[1]))
    return t


def _readable(t: torch.Tensor) -> torch.Tensor:
    """The operand with rows that the kernels can read in place: contiguous columns, 16-byte aligned base
    and, in 16 bits, rows (copied only where it has not)."""
    unit = 1 if t.dtype == torch.float32 else 8
    if (t.stride(1) != 1 and t.shape[1] > 1) or _ld(t) % unit or _ld(t) < t.shape[1]:
        t = t.contiguous()
    return _aligned(t)


class _GluFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, up, act):
        h, pre_gate, pre_up = _glu_forward(x, gate, up, act, True)
        ctx.save_for_backward(x, gate, up, pre_gate, pre_up)
        ctx.act = act
        return h if h.shape[1] == gate.shape[0] else h[:, : gate.shape[0]].contiguous()

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        x, gate, up, pre_gate, pre_up = ctx.saved_tensors
        need_x, need_g, need_u, _ = ctx.needs_input_grad
        dx, dw = _glu_backward(dh, x, gate, up, pre_gate, pre_up, ctx.act, need_x, need_g or need_u)
        ffn = gate.shape[0]
        return (dx, dw[:ffn] if need_g else None, dw[_round8(ffn):] if need_u else None, None)


@torch.library.custom_op("orda_b200::glu_forward", mutates_args=())
def _glu_forward_op(x: torch.Tensor, gate: torch.Tensor, up: torch.Tensor,
                    act: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    h, pre_gate, pre_up = _glu_forward(_readable(x), _readable(gate), _readable(up), act, True)
    return (h if h.shape[1] == gate.shape[0] else h[:, : gate.shape[0]].contiguous()), pre_gate, pre_up


@_glu_forward_op.register_fake
def _(x, gate, up, act):
    fp = (gate.shape[0] + 7) // 8 * 8
    return x.new_empty((x.shape[0], gate.shape[0])), x.new_empty((x.shape[0], fp)), x.new_empty((x.shape[0], fp))


@torch.library.custom_op("orda_b200::glu_backward", mutates_args=())
def _glu_backward_op(dh: torch.Tensor, x: torch.Tensor, gate: torch.Tensor, up: torch.Tensor, pre_gate: torch.Tensor,
                     pre_up: torch.Tensor, act: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    dx, dw = _glu_backward(dh, _readable(x), _readable(gate), _readable(up), pre_gate, pre_up, act, True, True)
    ffn = gate.shape[0]
    return dx, dw[:ffn].clone(), dw[_round8(ffn):].clone()  # an op's outputs share no storage


@_glu_backward_op.register_fake
def _(dh, x, gate, up, pre_gate, pre_up, act):
    return x.new_empty(x.shape), x.new_empty(gate.shape), x.new_empty(gate.shape)


def _glu_setup(ctx, inputs, output):
    x, gate, up, act = inputs
    ctx.save_for_backward(x, gate, up, output[1], output[2])
    ctx.act = act


def _glu_op_backward(ctx, dh, _dg, _du):
    return (*torch.ops.orda_b200.glu_backward(dh, *ctx.saved_tensors, ctx.act), None)


_glu_forward_op.register_autograd(_glu_op_backward, setup_context=_glu_setup)


def gated_linear_unit(x: torch.Tensor, gate_weight: torch.Tensor, up_weight: torch.Tensor, *,
                      activation: Activation = "silu") -> torch.Tensor:
    """``activation(x @ gate_weight.T) * (x @ up_weight.T)``, both products, the activation and the product
    of the two in one kernel.

    ``x`` is ``[..., hidden]``, the weights ``[ffn, hidden]``; the result is ``[..., ffn]``. ``activation``
    is ``"silu"``, ``"gelu"`` (erf), ``"gelu_tanh"`` or ``"relu"``. The compute dtype follows the loss's rule
    (active autocast dtype, else bf16 if any input is bf16, else fp16, else fp32); products and the
    activation are formed in fp32 and rounded once. fp32 runs on CUDA cores, exactly but without the tensor
    cores' speed. Back-propagates into all three; the backward pass keeps the two products in the compute
    dtype. Inputs with a hidden size that is no multiple of 8 are copied into padded rows first.
    """
    if activation not in _ACT_CODE:
        raise ValueError(f"activation must be one of {sorted(_ACT_CODE)}, got {activation!r}")
    if gate_weight.ndim != 2 or gate_weight.shape != up_weight.shape:
        raise ValueError(f"gate_weight and up_weight must have one shape (ffn, hidden), got "
                         f"{tuple(gate_weight.shape)} and {tuple(up_weight.shape)}")
    if x.ndim < 1 or x.shape[-1] != gate_weight.shape[1]:
        raise ValueError(f"x must have shape (..., {gate_weight.shape[1]}), got {tuple(x.shape)}")
    if 0 in gate_weight.shape:
        raise ValueError(f"gate_weight must not be empty, got shape={tuple(gate_weight.shape)}")
    for name, t in (("x", x), ("gate_weight", gate_weight), ("up_weight", up_weight)):
        if t.dtype not in _DTYPE_CODE:
            raise ValueError(f"{name} must be float32, float16 or bfloat16, got {t.dtype}")
    _require_cuda("gated_linear_unit", x, gate_weight, up_weight)
    dtype = default_compute_dtype(gate_weight, up_weight, x)
    act, ffn = _ACT_CODE[activation], gate_weight.shape[0]
    flat = _cast_padded(x if x.ndim == 2 else x.reshape(-1, x.shape[-1]), dtype)
    gate, up = _cast_padded(gate_weight, dtype), _cast_padded(up_weight, dtype)
    if torch.compiler.is_compiling():
        h = torch.ops.orda_b200.glu_forward(flat, gate, up, act)[0]
        return h if x.ndim == 2 else h.view(*x.shape[:-1], ffn)
    flat, gate, up = _readable(flat), _readable(gate), _readable(up)
    if torch.is_grad_enabled() and (flat.requires_grad or gate.requires_grad or up.requires_grad):
        h = _GluFunction.apply(flat, gate, up, act)
    else:
        h = _glu_forward(flat, gate, up, act, False)[0]
        h = h if h.shape[1] == ffn else h[:, :ffn].contiguous()
    return h if x.ndim == 2 else h.view(*x.shape[:-1], ffn)


# ------------------------------------------------------------------------------------------ rotary positions
@dataclass(frozen=True)
class RotaryConfig:
    """How positions turn the pairs of a head: pair ``i`` at position ``p`` by ``p * base^(-2 i / rotary_dim)``.

    * ``rotary_dim`` - the first ``rotary_dim`` elements of a head are rotated (``None``: all).
    * ``layout`` - ``"half"``: pairs ``(i, i + rotary_dim / 2)``; ``"interleaved"``: pairs ``(2 i, 2 i + 1)``.
    * ``scaling`` - contexts ``factor`` times as long: ``"linear"`` divides every angle by ``factor``;
      ``"ntk"`` raises ``base`` to ``base * factor^(d / (d - 2))``; ``"yarn"`` divides the angles of pairs
      that turn less than ``beta_slow`` times within ``original_positions``, keeps those that turn more than
      ``beta_fast`` times, blends in between, and multiplies the rotated values by
      ``0.1 ln(factor) + 1`` (or ``magnitude``).
    """

    head_dim: int
    rotary_dim: int | None = None
    base: float = 10000.0
    layout: Layout = "half"
    scaling: Scaling = "none"
    factor: float = 1.0
    original_positions: int = 4096
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    magnitude: float | None = None

    def __post_init__(self):
        if not 1 <= self.head_dim <= _native.ROTARY_MAX_DIM:
            raise ValueError(f"head_dim must be in 1 .. {_native.ROTARY_MAX_DIM}, got {self.head_dim}")
        d = self.head_dim if self.rotary_dim is None else self.rotary_dim
        if d % 2 or not 2 <= d <= self.head_dim:
            raise ValueError(f"rotary_dim must be even and in 2 .. head_dim={self.head_dim}, got {d}")
        if self.layout not in _LAYOUT_CODE:
            raise ValueError(f"layout must be 'half' or 'interleaved', got {self.layout!r}")
        if self.scaling not in ("none", "linear", "ntk", "yarn"):
            raise ValueError(f"scaling must be 'none', 'linear', 'ntk' or 'yarn', got {self.scaling!r}")
        if not (self.base > 0.0 and math.isfinite(self.base)):
            raise ValueError(f"base must be > 0, got {self.base}")
        if not (self.factor >= 1.0 and math.isfinite(self.factor)):
            raise ValueError(f"factor must be >= 1, got {self.factor}")
        if self.scaling == "ntk" and d == 2:
            raise ValueError("scaling='ntk' needs rotary_dim > 2")
        if self.scaling == "yarn" and not (self.beta_fast > self.beta_slow and self.original_positions > 0):
            raise ValueError("scaling='yarn' needs beta_fast > beta_slow and original_positions > 0")

    @property
    def dim(self) -> int:
        return self.head_dim if self.rotary_dim is None else self.rotary_dim

    def frequencies(self) -> list[float]:
        """Radians per position of each pair."""
        d, base = self.dim, self.base
        if self.scaling == "ntk":
            base *= self.factor ** (d / (d - 2))
        theta = [base ** (-2.0 * i / d) for i in range(d // 2)]
        if self.scaling == "linear":
            return [t / self.factor for t in theta]
        if self.scaling == "yarn":
            out = []
            for t in theta:
                turns = self.original_positions * t / (2.0 * math.pi)
                keep = min(1.0, max(0.0, (turns - self.beta_slow) / (self.beta_fast - self.beta_slow)))
                out.append(t / self.factor * (1.0 - keep) + t * keep)
            return out
        return theta

    @property
    def value_scale(self) -> float:
        """Factor of the rotated values."""
        if self.magnitude is not None:
            return float(self.magnitude)
        return 0.1 * math.log(self.factor) + 1.0 if self.scaling == "yarn" else 1.0

    def _key(self) -> tuple:
        return (tuple(self.frequencies()), self.head_dim, self.dim, _LAYOUT_CODE[self.layout], self.value_scale)


@lru_cache(maxsize=64)
def _rotary_plan(config: RotaryConfig):
    """(C array of the frequencies, its address, rotary_dim, layout code, magnitude): from the configuration alone."""
    f = config.frequencies()
    arr = (ctypes.c_double * len(f))(*f)
    return arr, ctypes.addressof(arr), config.dim, _LAYOUT_CODE[config.layout], config.value_scale


def _strides4(t: torch.Tensor) -> tuple[int, int, int]:
    s = t.stride()
    return (s[0], s[1], s[2]) if t.ndim == 4 else (0, s[0], s[1])


def _rotary_args(config, q, k, positions, out_q, out_k, inverse, weights=None, eps=0.0, dy=None, dweights=None):
    _arr, freq, rotary_dim, layout, magnitude = _rotary_plan(config)
    batch, seq = (q.shape[0], q.shape[1]) if q.ndim == 4 else (1, q.shape[0])
    ps = positions.stride()
    ps = ps if q.ndim == 4 else (0, ps[0])
    none2, zero6 = (None, None), (0,) * 6
    return _native.RotaryArgs(
        _native.ABI_VERSION, _DTYPE_CODE[q.dtype], batch, seq, (q.shape[-2], k.shape[-2]), config.head_dim, rotary_dim,
        layout, inverse,
        (q.data_ptr(), k.data_ptr()), (*_strides4(q), *_strides4(k)),
        (out_q.data_ptr(), out_k.data_ptr()), (*_strides4(out_q), *_strides4(out_k)),
        none2 if dy is None else (dy[0].data_ptr(), dy[1].data_ptr()),
        zero6 if dy is None else (*_strides4(dy[0]), *_strides4(dy[1])),
        positions.data_ptr(), ps, positions.dtype == torch.int64,
        _native.F32 if weights is None else _DTYPE_CODE[weights[0].dtype], freq, magnitude, eps,
        none2 if weights is None else (weights[0].data_ptr(), weights[1].data_ptr()),
        none2 if dweights is None else (dweights[0].data_ptr(), dweights[1].data_ptr()))


def _dense_last(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _new(t: torch.Tensor) -> torch.Tensor:
    return torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _rotate(q, k, positions, config, inverse: bool, weights=None, eps: float = 0.0):
    out_q, out_k = _new(q), _new(k)
    with _On(q.device) as stream:
        a = _rotary_args(config, q, k, positions, out_q, out_k, inverse, weights, eps)
        _native.check(_native.load().orda_rotary_forward(a, stream), "orda_rotary_forward")
    return out_q, out_k


def _norm_rotate_backward(dq, dk, q, k, weights, positions, config, eps: float):
    dq, dk = _dense_last(dq), _dense_last(dk)
    gq, gk = _new(q), _new(k)
    gw = (torch.empty_like(weights[0]), torch.empty_like(weights[1]))
    lib = _native.load()
    with _On(q.device) as stream:
        a = _rotary_args(config, q, k, positions, gq, gk, 0, weights, eps, (dq, dk), gw)
        size = int(lib.orda_qk_norm_rotary_backward_workspace_bytes(a))
        ws = torch.empty(max(size, 16), dtype=torch.uint8, device=q.device)
        _native.check(lib.orda_qk_norm_rotary_backward(a, ws.data_ptr(), size, stream), "orda_qk_norm_rotary_backward")
    return gq, gk, gw[0], gw[1]


class _RotaryFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, config):
        ctx.save_for_backward(positions)
        ctx.config = config
        return _rotate(q, k, positions, config, False)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        (positions,) = ctx.saved_tensors
        return (*_rotate(_dense_last(dq), _dense_last(dk), positions, ctx.config, True), None, None)


class _QkNormRotaryFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, config, eps):
        ctx.save_for_backward(q, k, q_weight, k_weight, positions)
        ctx.config, ctx.eps = config, eps
        return _rotate(q, k, positions, config, False, (q_weight, k_weight), eps)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        q, k, q_weight, k_weight, positions = ctx.saved_tensors
        return (*_norm_rotate_backward(dq, dk, q, k, (q_weight, k_weight), positions, ctx.config, ctx.eps),
                None, None, None)


# The custom ops that torch.compile traces take the configuration as plain values.
def _config_values(c: RotaryConfig):
    return [c.head_dim, c.dim, c.original_positions], [c.base, c.factor, c.beta_fast, c.beta_slow, c.value_scale], \
        c.layout, c.scaling


def _config_from(ints, floats, layout, scaling) -> RotaryConfig:
    return RotaryConfig(ints[0], ints[1], floats[0], layout, scaling, floats[1], ints[2], floats[2], floats[3], floats[4])


@torch.library.custom_op("orda_b200::rotary", mutates_args=())
def _rotary_op(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, q_weight: Optional[torch.Tensor],
               k_weight: Optional[torch.Tensor], eps: float, inverse: bool, ints: list[int], floats: list[float],
               layout: str, scaling: str) -> tuple[torch.Tensor, torch.Tensor]:
    config = _config_from(ints, floats, layout, scaling)
    weights = None if q_weight is None else (q_weight, k_weight)
    return _rotate(_dense_last(q), _dense_last(k), positions, config, inverse, weights, eps)


@_rotary_op.register_fake
def _(q, k, positions, q_weight, k_weight, eps, inverse, ints, floats, layout, scaling):
    return q.new_empty(q.shape), k.new_empty(k.shape)


@torch.library.custom_op("orda_b200::qk_norm_rotary_backward", mutates_args=())
def _qk_norm_rotary_backward_op(dq: torch.Tensor, dk: torch.Tensor, q: torch.Tensor, k: torch.Tensor,
                                positions: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, eps: float,
                                ints: list[int], floats: list[float], layout: str,
                                scaling: str) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    return _norm_rotate_backward(dq, dk, _dense_last(q), _dense_last(k), (q_weight, k_weight), positions,
                                 _config_from(ints, floats, layout, scaling), eps)


@_qk_norm_rotary_backward_op.register_fake
def _(dq, dk, q, k, positions, q_weight, k_weight, eps, ints, floats, layout, scaling):
    return q.new_empty(q.shape), k.new_empty(k.shape), q_weight.new_empty(q_weight.shape), k_weight.new_empty(k_weight.shape)


def _rotary_setup(ctx, inputs, output):
    q, k, positions, q_weight, k_weight, eps, inverse, ints, floats, layout, scaling = inputs
    ctx.normed, ctx.eps, ctx.inverse, ctx.config = q_weight is not None, eps, inverse, (ints, floats, layout, scaling)
    ctx.save_for_backward(positions, *((q, k, q_weight, k_weight) if ctx.normed else ()))


def _rotary_op_backward(ctx, dq, dk):
    if ctx.normed:
        positions, q, k, q_weight, k_weight = ctx.saved_tensors
        gq, gk, gwq, gwk = torch.ops.orda_b200.qk_norm_rotary_backward(dq, dk, q, k, positions, q_weight, k_weight,
                                                                       ctx.eps, *ctx.config)
        return (gq, gk, None, gwq, gwk, *([None] * 6))
    gq, gk = torch.ops.orda_b200.rotary(dq, dk, ctx.saved_tensors[0], None, None, 0.0, not ctx.inverse, *ctx.config)
    return (gq, gk, *([None] * 9))


_rotary_op.register_autograd(_rotary_op_backward, setup_context=_rotary_setup)


def _check_qk(what: str, q, k, positions, config):
    if not isinstance(config, RotaryConfig):
        raise TypeError(f"{what}: config must be a RotaryConfig, got {type(config).__name__}")
    if q.ndim not in (3, 4) or k.ndim != q.ndim or q.shape[:-2] != k.shape[:-2]:
        raise ValueError(f"{what}: q and k must be (batch, seq, heads, head_dim) or (tokens, heads, head_dim) with the "
                         f"same tokens, got {tuple(q.shape)} and {tuple(k.shape)}")
    if q.shape[-1] != config.head_dim or k.shape[-1] != config.head_dim:
        raise ValueError(f"{what}: heads must have config.head_dim={config.head_dim} elements, got {q.shape[-1]} and "
                         f"{k.shape[-1]}")
    if q.dtype not in _DTYPE_CODE or k.dtype != q.dtype:
        raise ValueError(f"{what}: q and k must both be float32, float16 or bfloat16, got {q.dtype} and {k.dtype}")
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{what}: positions must be int32 or int64, got {positions.dtype}")
    if positions.shape != q.shape[:-2] and positions.shape != q.shape[-3:-2]:
        raise ValueError(f"{what}: positions must have shape {tuple(q.shape[:-2])} or {tuple(q.shape[-3:-2])}, got "
                         f"{tuple(positions.shape)}")
    if q.ndim == 4 and positions.ndim == 1:
        positions = positions.expand(q.shape[0], q.shape[1])
    return positions


def rotary_embedding(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor,
                     config: RotaryConfig) -> tuple[torch.Tensor, torch.Tensor]:
    """Queries and keys with their positions rotated in, as new contiguous tensors, in one pass.

    ``q`` is ``[batch, seq, q_heads, head_dim]`` or ``[tokens, q_heads, head_dim]`` and ``k`` alike with its
    own number of heads; any strides whose last is 1 are read in place (slices of a fused projection,
    transposed ``[batch, heads, seq, head_dim]`` storage). ``positions`` are integers, ``[batch, seq]`` or
    ``[seq]`` (``[tokens]``), in any order, negative ones too; angles are formed in 64 bits, so far
    positions lose nothing. Back-propagates into ``q`` and ``k``.
    """
    positions = _check_qk("rotary_embedding", q, k, positions, config)
    _require_cuda("rotary_embedding", q, k, positions)
    if torch.compiler.is_compiling():
        return torch.ops.orda_b200.rotary(q, k, positions, None, None, 0.0, False, *_config_values(config))
    q, k = _dense_last(q), _dense_last(k)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad):
        return _RotaryFunction.apply(q, k, positions, config)
    return _rotate(q, k, positions, config, False)


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                   positions: torch.Tensor, config: RotaryConfig, eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """:func:`rotary_embedding` of ``q_weight * q / sqrt(mean(q^2) + eps)`` and the same of ``k``, each head
    normalised on its own, in the same pass (statistics in fp32, one rounding).

    The weights are ``[head_dim]``, both of one floating dtype. Back-propagates into all four; the weights'
    gradients are summed over tokens and heads in a fixed order.
    """
    what = "qk_norm_rotary"
    positions = _check_qk(what, q, k, positions, config)
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w.shape != (config.head_dim,):
            raise ValueError(f"{what}: {name} must have shape ({config.head_dim},), got {tuple(w.shape)}")
        if w.dtype not in _DTYPE_CODE or w.dtype != q_weight.dtype:
            raise ValueError(f"{what}: weights must have one dtype of float32, float16 and bfloat16, got "
                             f"{q_weight.dtype} and {k_weight.dtype}")
    if not eps >= 0.0:
        raise ValueError(f"{what}: eps must be >= 0, got {eps}")
    _require_cuda(what, q, k, positions, q_weight, k_weight)
    q_weight, k_weight = q_weight.contiguous(), k_weight.contiguous()
    if torch.compiler.is_compiling():
        return torch.ops.orda_b200.rotary(q, k, positions, q_weight, k_weight, float(eps), False,
                                          *_config_values(config))
    q, k = _dense_last(q), _dense_last(k)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or q_weight.requires_grad
                                    or k_weight.requires_grad):
        return _QkNormRotaryFunction.apply(q, k, q_weight, k_weight, positions, config, float(eps))
    return _rotate(q, k, positions, config, False, (q_weight, k_weight), float(eps))


# ------------------------------------------------------------------------------------------ gradient norm and clipping
def _dense(t: torch.Tensor) -> bool:
    """Whether the tensor's values fill one gapless stretch of memory (in any order of dimensions)."""
    if t.is_contiguous():
        return True
    expect = 1
    for size, stride in sorted(zip(t.shape, t.stride()), key=lambda p: p[1]):
        if size == 1:
            continue
        if stride != expect:
            return False
        expect *= size
    return True


def _check_gradients(what: str, tensors: Sequence[torch.Tensor]) -> None:
    for t in tensors:
        if t.dtype not in _DTYPE_CODE:
            raise ValueError(f"{what}: gradients must be float32, float16 or bfloat16, got {t.dtype}")
        if t.layout != torch.strided:
            raise ValueError(f"{what}: gradients must be strided tensors, got {t.layout}")
    if tensors:
        _require_cuda(what, *tensors)


def _clip_call(src: Sequence[torch.Tensor], dst: Sequence[torch.Tensor] | None, max_norm: float, eps: float):
    """The norm (0-dim fp32 tensor) of `src`; `dst` receives the clipped values. All dense, one device."""
    n = len(src)
    dev = src[0].device
    lib = _native.load()
    addresses = (ctypes.c_void_p * n)(*[t.data_ptr() for t in src])
    a = _native.TensorList(
        _native.ABI_VERSION, n, addresses,
        None if dst is None else addresses if dst is src else (ctypes.c_void_p * n)(*[t.data_ptr() for t in dst]),
        (ctypes.c_int64 * n)(*[t.numel() for t in src]), (ctypes.c_int32 * n)(*[_DTYPE_CODE[t.dtype] for t in src]))
    with _On(dev) as stream:
        norm = torch.empty((), dtype=torch.float32, device=dev)
        size = int(lib.orda_clip_workspace_bytes(a))
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        _native.check(lib.orda_clip_gradients(a, max_norm, eps, norm.data_ptr(), ws.data_ptr(), size, stream),
                      "orda_clip_gradients")
    return norm


def _check_clip(what: str, max_norm, eps) -> tuple[float, float]:
    max_norm, eps = float(max_norm), float(eps)
    if not max_norm >= 0.0:
        raise ValueError(f"{what}: max_norm must be >= 0, got {max_norm}")
    if not eps >= 0.0:
        raise ValueError(f"{what}: eps must be >= 0, got {eps}")
    return max_norm, eps


def grad_norm(gradients: Iterable[torch.Tensor]) -> torch.Tensor:
    """The 2-norm over all values of all tensors, as a 0-dim fp32 tensor on their device (squares are added
    in 64 bits, in a fixed order). No synchronisation."""
    src = [g.detach() for g in gradients]
    _check_gradients("grad_norm", src)
    if not src:
        return torch.zeros(())
    return _clip_call([g if _dense(g) else g.contiguous() for g in src], None, 0.0, 0.0)


def clip_gradients(gradients: Iterable[torch.Tensor], max_norm: float, *,
                   eps: float = 1e-6) -> tuple[list[torch.Tensor], torch.Tensor]:
    """``(clipped, norm)``: new tensors ``g * min(1, max_norm / (norm + eps))`` and the norm over all of them
    before clipping (0-dim fp32). The gradients themselves stay as they are. A norm that is infinite or
    NaN passes into the values, as in ``torch.nn.utils.clip_grad_norm_``. No synchronisation."""
    what = "clip_gradients"
    max_norm, eps = _check_clip(what, max_norm, eps)
    src = [g.detach() for g in gradients]
    _check_gradients(what, src)
    if not src:
        return [], torch.zeros(())
    src = [g if _dense(g) else g.contiguous() for g in src]
    out = [torch.empty_like(g) for g in src]  # dense: the same strides
    return out, _clip_call(src, out, max_norm, eps)


def clip_grad_norm_(parameters: torch.Tensor | Iterable[torch.Tensor], max_norm: float, *, eps: float = 1e-6,
                    error_if_nonfinite: bool = False) -> torch.Tensor:
    """``torch.nn.utils.clip_grad_norm_`` for the 2-norm: scales the ``.grad`` of every parameter in place by
    ``min(1, max_norm / (norm + eps))`` and returns the norm (0-dim fp32). Parameters without a gradient are
    skipped; gradients may have different dtypes and strides but must lie on one device, and no two may
    share memory (a parameter given twice is refused). Only ``error_if_nonfinite`` synchronises: it raises
    before anything is scaled."""
    what = "clip_grad_norm_"
    max_norm, eps = _check_clip(what, max_norm, eps)
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [p.grad.detach() for p in parameters if p.grad is not None]
    _check_gradients(what, grads)
    if not grads:
        return torch.zeros(())
    seen = set()
    for g in grads:
        if g.numel():
            if g.data_ptr() in seen:
                raise ValueError(f"{what}: a gradient appears twice among the parameters")
            seen.add(g.data_ptr())
    dense = [g if _dense(g) else g.contiguous() for g in grads]
    if error_if_nonfinite:
        norm = _clip_call(dense, None, 0.0, 0.0)
        if not math.isfinite(float(norm)):
            raise RuntimeError(f"{what}: the total norm of the gradients is {float(norm)}; with "
                               "error_if_nonfinite=False they are scaled by it all the same")
    norm = _clip_call(dense, dense, max_norm, eps)
    for g, d in zip(grads, dense):
        if d is not g:
            g.copy_(d)
    return norm


__all__ = [
    "RotaryConfig",
    "clip_grad_norm_",
    "clip_gradients",
    "gated_linear_unit",
    "grad_norm",
    "qk_norm_rotary",
    "rotary_embedding",
]
