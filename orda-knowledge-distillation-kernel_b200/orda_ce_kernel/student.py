"""Operators of a student's training step around :func:`orda_ce_kernel.distillation_loss`, and of its
token-by-token run (``include/orda_b200_student.h``; the reference leaves them to PyTorch, as the model
and training loop of ``test/benchmark/src/core.py:106-138`` and ``_train.py:102-452`` do):

* :func:`gated_linear_unit` - the gated feed-forward block ``act(x Wg^T) * (x Wu^T)`` in one kernel;
* :func:`rotary_embedding` - positions rotated into queries and keys in one pass;
* :func:`qk_norm_rotary` - per-head RMS norms of queries and keys, rotated in the same pass;
* :func:`grad_norm`, :func:`clip_gradients`, :func:`clip_grad_norm_` - the global gradient norm and clipping.

The first three back-propagate (once; no double backward, no forward-mode derivative: an input that carries a
tangent is refused) and become one custom op each under ``torch.compile`` and whatever else records calls
(``make_fx``, ``torch.jit.trace``, dispatch modes); the last three refuse to be recorded into a graph. As for
the loss there is no CPU fallback: CUDA tensors on a B200 are required. Every call runs on the current stream of
its tensors' device, takes its workspace from the caching allocator and does not synchronise, so it can be
captured into a CUDA graph; a captured backward pass is refused while an eager autograd graph of the default
stream still holds one of its leaves (a compiled one is PyTorch's own node, and is not: drop such graphs first).
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Iterable, Literal, Optional

import torch

from . import _native
from ._runtime import default_compute_dtype

Activation = Literal["silu", "gelu", "gelu_tanh", "relu"]
Layout = Literal["half", "interleaved"]
Scaling = Literal["none", "linear", "ntk", "yarn"]
Ramp = Literal["turns", "index"]

_LAYOUTS = ("half", "interleaved")
_DTYPES = (torch.float32, torch.float16, torch.bfloat16)
_binding = None


def _bound():
    """The extension module that holds the calls' host side; raises RuntimeError if it is not built."""
    global _binding
    if _binding is None:
        _native.load()
        try:
            from . import _student
        except ImportError as exc:
            raise RuntimeError("orda_ce_kernel/_student.so is not built for this torch (run "
                               f"orda-knowledge-distillation-kernel_b200/build.py --force): {exc}") from exc
        _binding = _student
    return _binding


# ------------------------------------------------------------------------------------------ gated feed-forward block
# The custom ops that torch.compile traces: the same launches, with autograd formulas over ops.
@torch.library.custom_op("orda_b200::glu_forward", mutates_args=())
def _glu_forward_op(x: torch.Tensor, gate: torch.Tensor, up: torch.Tensor, act: int) -> tuple[torch.Tensor, torch.Tensor]:
    return _bound().glu_forward(x, gate, up, act)


@_glu_forward_op.register_fake
def _(x, gate, up, act):
    rows = x.numel() // x.shape[-1]
    return x.new_empty((*x.shape[:-1], gate.shape[0])), x.new_empty((2, rows, (gate.shape[0] + 7) // 8 * 8))


@torch.library.custom_op("orda_b200::glu_backward", mutates_args=())
def _glu_backward_op(dh: torch.Tensor, x: torch.Tensor, gate: torch.Tensor, up: torch.Tensor, pre: torch.Tensor,
                     act: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return _bound().glu_backward(dh, x, gate, up, pre, act)


@_glu_backward_op.register_fake
def _(dh, x, gate, up, pre, act):
    return x.new_empty(x.shape), x.new_empty(gate.shape), x.new_empty(gate.shape)


def _glu_setup(ctx, inputs, output):
    x, gate, up, act = inputs
    ctx.save_for_backward(x, gate, up, output[1])
    ctx.act = act


def _glu_op_backward(ctx, dh, _dpre):
    _bound().refuse_eager_nodes_in_capture("gated_linear_unit")
    return (*torch.ops.orda_b200.glu_backward(dh, *ctx.saved_tensors, ctx.act), None)


_glu_forward_op.register_autograd(_glu_op_backward, setup_context=_glu_setup)

_ACT_CODE = {"silu": _native.ACT_SILU, "gelu": _native.ACT_GELU, "gelu_tanh": _native.ACT_GELU_TANH,
             "relu": _native.ACT_RELU}


def gated_linear_unit(x: torch.Tensor, gate_weight: torch.Tensor, up_weight: torch.Tensor, *,
                      activation: Activation = "silu") -> torch.Tensor:
    """``activation(x @ gate_weight.T) * (x @ up_weight.T)``, both products, the activation and the product
    of the two in one kernel.

    ``x`` is ``[..., hidden]``, the weights ``[ffn, hidden]``; the result is ``[..., ffn]``. ``activation``
    is ``"silu"``, ``"gelu"`` (erf), ``"gelu_tanh"`` or ``"relu"``. The compute dtype follows the loss's rule
    (active autocast dtype, else bf16 if any input is bf16, else fp16, else fp32); products and the
    activation are formed in fp32 and rounded once. fp32 runs on CUDA cores, without the tensor cores' speed (and
    slower than ``torch.nn.Linear``). Back-propagates into all three; the backward pass keeps the two products,
    and multiplies their gradients, in the compute dtype. Inputs with a hidden size that is no multiple of 8 are copied into padded rows first.
    """
    h = None
    if not torch.compiler.is_compiling():
        h = (_binding or _bound()).gated_linear_unit(x, gate_weight, up_weight, activation)
    if h is None:  # recorded: through the custom op
        if activation not in _ACT_CODE:
            raise ValueError(f"activation must be one of {sorted(_ACT_CODE)}, got {activation!r}")
        for t in (x, gate_weight, up_weight):
            if t.dtype not in _DTYPES:
                raise ValueError(f"gated_linear_unit: tensors must be float32, float16 or bfloat16, got {t.dtype}")
        dtype = default_compute_dtype(gate_weight, up_weight, x)
        h = torch.ops.orda_b200.glu_forward(x.to(dtype), gate_weight.to(dtype), up_weight.to(dtype),
                                            _ACT_CODE[activation])[0]
    return h


# ------------------------------------------------------------------------------------------ rotary positions
@dataclass(frozen=True)
class RotaryConfig:
    """How positions turn the pairs of a head: pair ``i`` at position ``p`` by ``p * base^(-2 i / rotary_dim)``.

    * ``rotary_dim`` - the first ``rotary_dim`` elements of a head are rotated (``None``: all).
    * ``layout`` - ``"half"``: pairs ``(i, i + rotary_dim / 2)``; ``"interleaved"``: pairs ``(2 i, 2 i + 1)``.
    * ``scaling`` - contexts ``factor`` times as long: ``"linear"`` divides every angle by ``factor``;
      ``"ntk"`` raises ``base`` to ``base * factor^(d / (d - 2))``; ``"yarn"`` divides the angles of pairs
      that turn less than ``beta_slow`` times within ``original_positions``, keeps those that turn more than
      ``beta_fast`` times, blends in between (``ramp``), and multiplies the rotated values by
      ``0.1 ln(factor) + 1`` (or ``magnitude``).
    * ``ramp`` - the part of a pair's own angle in YaRN's blend. ``"turns"``: linear in its turns within
      ``original_positions``, 0 at ``beta_slow`` and 1 at ``beta_fast``, as the paper has it. ``"index"``: linear
      in the pair's index ``i``, 1 up to the last pair that turns ``beta_fast`` times and 0 from the first that
      turns ``beta_slow`` times or less, as published checkpoints mostly have it. The two differ by up to 57% in a
      pair's angle (128 elements, factor 8), so a checkpoint needs the one it was trained with.
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
    ramp: Ramp = "turns"

    def __post_init__(self):
        if not 1 <= self.head_dim <= _native.ROTARY_MAX_DIM:
            raise ValueError(f"head_dim must be in 1 .. {_native.ROTARY_MAX_DIM}, got {self.head_dim}")
        d = self.head_dim if self.rotary_dim is None else self.rotary_dim
        if d % 2 or not 2 <= d <= self.head_dim:
            raise ValueError(f"rotary_dim must be even and in 2 .. head_dim={self.head_dim}, got {d}")
        if self.layout not in _LAYOUTS:
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
        if self.ramp not in ("turns", "index"):
            raise ValueError(f"ramp must be 'turns' or 'index', got {self.ramp!r}")
        if self.scaling == "yarn" and self.ramp == "index" and not (self.base > 1.0 and self.beta_slow > 0.0):
            raise ValueError("scaling='yarn' with ramp='index' needs base > 1 and beta_slow > 0")
        object.__setattr__(self, "_plan", None)

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
            return [t / self.factor * (1.0 - keep) + t * keep for t, keep in zip(theta, self._kept(theta))]
        return theta

    def _kept(self, theta: list[float]) -> list[float]:
        """YaRN: the part of each pair's own angle in the blend."""
        if self.ramp == "turns":
            def at(i):
                return self.original_positions * theta[i] / (2.0 * math.pi)

            slow, fast = self.beta_slow, self.beta_fast
        else:
            def index(turns):  # of the pair that turns so often; not a whole number
                return self.dim * math.log(self.original_positions / (2.0 * math.pi * turns)) / (2.0 * math.log(self.base))

            def at(i):
                return i

            fast, slow = max(0, math.floor(index(self.beta_fast))), min(self.dim - 1, math.ceil(index(self.beta_slow)))
            if slow <= 0:  # no pair turns that often
                return [0.0] * len(theta)
            if slow <= fast:
                slow = fast + 0.001  # a step
        return [min(1.0, max(0.0, (at(i) - slow) / (fast - slow))) for i in range(len(theta))]

    @property
    def value_scale(self) -> float:
        """Factor of the rotated values."""
        if self.magnitude is not None:
            return float(self.magnitude)
        return 0.1 * math.log(self.factor) + 1.0 if self.scaling == "yarn" else 1.0

    def __getstate__(self):
        return self.__dict__ | {"_plan": None}  # the plan is rebuilt where it is used


def _plan(config: RotaryConfig):
    """The configuration in the binding's form, built once per configuration object."""
    if config._plan is None:
        object.__setattr__(config, "_plan", _bound().RotaryPlan(config.frequencies(), config.head_dim,
                                                               config.layout == "interleaved", config.value_scale))
    return config._plan


# The custom ops take the configuration as plain values.
def _config_values(c: RotaryConfig):
    return [c.head_dim, c.dim, c.original_positions], [c.base, c.factor, c.beta_fast, c.beta_slow, c.value_scale], \
        c.layout, c.scaling, c.ramp


def _config_from(ints, floats, layout, scaling, ramp) -> RotaryConfig:
    return RotaryConfig(ints[0], ints[1], floats[0], layout, scaling, floats[1], ints[2], floats[2], floats[3], floats[4],
                        ramp)


@torch.library.custom_op("orda_b200::rotary", mutates_args=())
def _rotary_op(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, q_weight: Optional[torch.Tensor],
               k_weight: Optional[torch.Tensor], eps: float, inverse: bool, ints: list[int], floats: list[float],
               layout: str, scaling: str, ramp: str) -> tuple[torch.Tensor, torch.Tensor]:
    plan = _plan(_config_from(ints, floats, layout, scaling, ramp))
    return _bound().rotary(q, k, positions, q_weight, k_weight, eps, inverse, plan)


@_rotary_op.register_fake
def _(q, k, positions, q_weight, k_weight, eps, inverse, ints, floats, layout, scaling, ramp):
    return q.new_empty(q.shape), k.new_empty(k.shape)


@torch.library.custom_op("orda_b200::qk_norm_rotary_backward", mutates_args=())
def _qk_norm_rotary_backward_op(dq: torch.Tensor, dk: torch.Tensor, q: torch.Tensor, k: torch.Tensor,
                                positions: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, eps: float,
                                ints: list[int], floats: list[float], layout: str, scaling: str,
                                ramp: str) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    plan = _plan(_config_from(ints, floats, layout, scaling, ramp))
    return _bound().qk_norm_rotary_backward(dq, dk, q, k, positions, q_weight, k_weight, eps, plan)


@_qk_norm_rotary_backward_op.register_fake
def _(dq, dk, q, k, positions, q_weight, k_weight, eps, ints, floats, layout, scaling, ramp):
    return q.new_empty(q.shape), k.new_empty(k.shape), q_weight.new_empty(q_weight.shape), k_weight.new_empty(k_weight.shape)


def _rotary_setup(ctx, inputs, output):
    q, k, positions, q_weight, k_weight, eps, inverse, *config = inputs
    ctx.normed, ctx.eps, ctx.inverse, ctx.config = q_weight is not None, eps, inverse, config
    ctx.save_for_backward(positions, *((q, k, q_weight, k_weight) if ctx.normed else ()))


def _rotary_op_backward(ctx, dq, dk):
    _bound().refuse_eager_nodes_in_capture("qk_norm_rotary" if ctx.normed else "rotary_embedding")
    if ctx.normed:
        positions, q, k, q_weight, k_weight = ctx.saved_tensors
        gq, gk, gwq, gwk = torch.ops.orda_b200.qk_norm_rotary_backward(dq, dk, q, k, positions, q_weight, k_weight,
                                                                       ctx.eps, *ctx.config)
        return (gq, gk, None, gwq, gwk, *([None] * 7))
    gq, gk = torch.ops.orda_b200.rotary(dq, dk, ctx.saved_tensors[0], None, None, 0.0, not ctx.inverse, *ctx.config)
    return (gq, gk, *([None] * 10))


_rotary_op.register_autograd(_rotary_op_backward, setup_context=_rotary_setup)


def _require_config(what: str, config) -> None:
    if not isinstance(config, RotaryConfig):
        raise TypeError(f"{what}: config must be a RotaryConfig, got {type(config).__name__}")


def rotary_embedding(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor,
                     config: RotaryConfig) -> tuple[torch.Tensor, torch.Tensor]:
    """Queries and keys with their positions rotated in, as new contiguous tensors, in one pass.

    ``q`` is ``[batch, seq, q_heads, head_dim]`` or ``[tokens, q_heads, head_dim]`` and ``k`` alike with its
    own number of heads; any strides whose last is 1 are read in place (slices of a fused projection,
    transposed ``[batch, heads, seq, head_dim]`` storage). ``positions`` are integers, ``[batch, seq]`` or
    ``[seq]`` (``[tokens]``), in any order, negative ones too; angles are formed in 64 bits, so far
    positions lose nothing. Back-propagates into ``q`` and ``k``.
    """
    _require_config("rotary_embedding", config)
    out = None
    if not torch.compiler.is_compiling():
        out = (_binding or _bound()).rotary_embedding(q, k, positions, config._plan or _plan(config))
    if out is None:  # recorded: through the custom op
        out = torch.ops.orda_b200.rotary(q, k, positions, None, None, 0.0, False, *_config_values(config))
    return out


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                   positions: torch.Tensor, config: RotaryConfig, eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """:func:`rotary_embedding` of ``q_weight * q / sqrt(mean(q^2) + eps)`` and the same of ``k``, each head
    normalised on its own, in the same pass (statistics in fp32, one rounding).

    The weights are ``[head_dim]``, both of one floating dtype. Back-propagates into all four; the weights'
    gradients are summed over tokens and heads in a fixed order.
    """
    _require_config("qk_norm_rotary", config)
    out = None
    if not torch.compiler.is_compiling():
        out = (_binding or _bound()).qk_norm_rotary(q, k, q_weight, k_weight, positions, config._plan or _plan(config), eps)
    if out is None:  # recorded: through the custom op
        out = torch.ops.orda_b200.rotary(q, k, positions, q_weight, k_weight, float(eps), False,
                                         *_config_values(config))
    return out


# ------------------------------------------------------------------------------------------ gradient norm and clipping
def grad_norm(gradients: Iterable[torch.Tensor]) -> torch.Tensor:
    """The 2-norm over all values of all tensors, as a 0-dim fp32 tensor on their device (squares are added
    in 64 bits, in a fixed order). No synchronisation."""
    return (_binding or _bound()).grad_norm(list(gradients))


def clip_gradients(gradients: Iterable[torch.Tensor], max_norm: float, *,
                   eps: float = 1e-6) -> tuple[list[torch.Tensor], torch.Tensor]:
    """``(clipped, norm)``: new tensors ``g * min(1, max_norm / (norm + eps))`` and the norm over all of them
    before clipping (0-dim fp32). The gradients themselves stay as they are. Results of up to 16 MiB in all
    share one allocation. A norm that is infinite or
    NaN passes into the values, as in ``torch.nn.utils.clip_grad_norm_``. No synchronisation."""
    return (_binding or _bound()).clip_gradients(list(gradients), max_norm, eps)


def clip_grad_norm_(parameters: torch.Tensor | Iterable[torch.Tensor], max_norm: float, *, eps: float = 1e-6,
                    error_if_nonfinite: bool = False) -> torch.Tensor:
    """``torch.nn.utils.clip_grad_norm_`` for the 2-norm: scales the ``.grad`` of every parameter in place by
    ``min(1, max_norm / (norm + eps))`` and returns the norm (0-dim fp32). Parameters without a gradient are
    skipped; gradients may have different dtypes and strides but must lie on one device, and no two may
    share memory (refused, as is a parameter given twice, and a gradient that holds broadcast values). Only ``error_if_nonfinite`` synchronises: it raises
    before anything is scaled."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [p.grad for p in parameters if p.grad is not None]
    if error_if_nonfinite:
        norm = float(grad_norm(grads))
        if not math.isfinite(norm):
            raise RuntimeError(f"clip_grad_norm_: the total norm of the gradients is {norm}; with "
                               "error_if_nonfinite=False they are scaled by it all the same")
    return (_binding or _bound()).clip_in_place(grads, max_norm, eps)


__all__ = [
    "RotaryConfig",
    "clip_grad_norm_",
    "clip_gradients",
    "gated_linear_unit",
    "grad_norm",
    "qk_norm_rotary",
    "rotary_embedding",
]
