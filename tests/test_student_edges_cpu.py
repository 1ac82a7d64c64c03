"""``orda_ce_kernel.student`` without a GPU, at the edges: refusals that keep a kernel from reading behind a
tensor, and what the calls do while something traces them."""
from __future__ import annotations

import pytest
import torch

from orda_ce_kernel import _native, student

OPS = torch.ops.orda_b200


# ------------------------------------------------------------------------------------------ custom ops
def _glu_backward(**change):
    a = dict(dh=torch.randn(2, 3, 13), x=torch.randn(2, 3, 8), gate=torch.randn(13, 8), up=torch.randn(13, 8),
             pre=torch.randn(2, 6, 16), act=0) | change
    return OPS.glu_backward(*a.values())


@pytest.mark.parametrize("change,match", [
    (dict(pre=torch.randn(2, 6, 13)), "products"), (dict(pre=torch.randn(2, 5, 16)), "products"),
    (dict(pre=torch.randn(2, 6, 16).half()), "products"), (dict(pre=torch.randn(192)), "products"),
    (dict(dh=torch.randn(2, 3, 12)), "gradient"), (dict(dh=torch.randn(2, 2, 13)), "gradient"),
    (dict(dh=torch.randn(2, 3, 13).bfloat16()), "gradient"), (dict(up=torch.randn(12, 8)), "one shape"),
])
def test_glu_backward_op_refuses_tensors_of_other_sizes(change, match):
    with pytest.raises(ValueError, match=match):
        _glu_backward(**change)


def test_well_formed_custom_ops_reach_the_device_check():
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        _glu_backward()
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        _norm_backward()


def _norm_backward(**change):
    q, k, w = torch.randn(4, 2, 8), torch.randn(4, 1, 8), torch.ones(8)
    a = dict(dq=q, dk=k, q=q, k=k, positions=torch.arange(4), q_weight=w, k_weight=w, eps=1e-6) | change
    return OPS.qk_norm_rotary_backward(*a.values(), *student._config_values(student.RotaryConfig(8)))


@pytest.mark.parametrize("change,match", [
    (dict(dq=torch.randn(3, 2, 8)), "queries"), (dict(dq=torch.randn(4, 1, 8)), "queries"),
    (dict(dk=torch.randn(4, 1, 6)), "keys"), (dict(dk=torch.randn(4, 1, 8).half()), "keys"),
])
def test_norm_backward_op_refuses_gradients_of_other_sizes(change, match):
    with pytest.raises(ValueError, match=match):
        _norm_backward(**change)


def test_rotary_op_refuses_one_weight():
    q, k, cfg = torch.randn(4, 2, 8), torch.randn(4, 1, 8), student._config_values(student.RotaryConfig(8))
    for weights in ((torch.ones(8), None), (None, torch.ones(8))):
        with pytest.raises(ValueError, match="together"):
            OPS.rotary(q, k, torch.arange(4), *weights, 1e-6, False, *cfg)


# ------------------------------------------------------------------------------------------ sizes
@pytest.mark.parametrize("heads", [2 ** 29 + 1, 2 ** 31, 2 ** 32 + 1])
def test_head_counts_that_do_not_fit_are_refused(heads):
    """Heads are counted in 32 bits: 2^32 + 1 broadcast heads must not become one."""
    one, many, pos = torch.randn(4, 1, 8), torch.randn(4, 1, 8).expand(4, heads, 8), torch.arange(4)
    cfg, w = student.RotaryConfig(8), torch.ones(8)
    for q, k in ((many, one), (one, many)):
        with pytest.raises(ValueError, match="heads each"):
            student.rotary_embedding(q, k, pos, cfg)
        with pytest.raises(ValueError, match="heads each"):
            student.qk_norm_rotary(q, k, w, w, pos, cfg)


def test_c_head_counts_are_bounded():
    lib = _native.load()
    for heads in ((2 ** 29 + 1, 1), (1, 2 ** 29 + 1), (2 ** 31 - 1, 2 ** 31 - 1)):
        a = _native.RotaryArgs(abi_version=_native.ABI_VERSION, dtype=_native.BF16, batch=1, seq=1, heads=heads, head_dim=8,
                               rotary_dim=0, x=(16, 16), out=(16, 16), positions=16, magnitude=1.0)
        assert lib.orda_rotary_forward(a, None) == _native.ERR_UNSUPPORTED


# ------------------------------------------------------------------------------------------ clipping in place
def _clip(*grads):
    params = []
    for g in grads:
        p = torch.nn.Parameter(torch.empty(g.shape, dtype=g.dtype))
        p.grad = g
        params.append(p)
    return student.clip_grad_norm_(params, 1.0)


def test_clip_refuses_gradients_that_share_memory():
    flat = torch.ones(100)
    for grads, match in (((flat[:60], flat[59:]), "share memory"), ((flat[10:20], flat), "share memory"),
                         ((flat, flat[50:60], torch.ones(3)), "share memory"), ((flat, flat), "twice"),
                         ((flat[::2], flat[::2]), "twice"), ((torch.ones(1, 8).expand(4, 8),), "broadcast"),
                         ((torch.ones(3), torch.ones(()).expand(5)), "broadcast")):
        with pytest.raises(ValueError, match=match):
            _clip(*grads)
    for grads in ((flat[:60], flat[60:]), (flat[::2], flat[1::2]), (flat[:50].view(5, 10).T, flat[50:]), (flat[:0], flat[:0])):
        with pytest.raises(RuntimeError, match="no CPU fallback"):  # well-formed
            _clip(*grads)


# ------------------------------------------------------------------------------------------ tangents and recorders
def test_inputs_that_carry_a_tangent_are_refused():
    """A result without one would count as a constant."""
    from torch.autograd import forward_ad

    x, w, v, pos, cfg = torch.randn(4, 2, 8), torch.randn(12, 8), torch.ones(8), torch.arange(4), student.RotaryConfig(8)
    g = torch.ones(3)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        p = torch.nn.Parameter(torch.ones(3))
        p.grad = dual(g)
        for call in (lambda: student.gated_linear_unit(dual(x), w, w), lambda: student.gated_linear_unit(x, dual(w), w),
                     lambda: student.gated_linear_unit(x, w, dual(w)), lambda: student.rotary_embedding(dual(x), x, pos, cfg),
                     lambda: student.rotary_embedding(x, dual(x), pos, cfg),
                     lambda: student.qk_norm_rotary(dual(x), x, v, v, pos, cfg),
                     lambda: student.qk_norm_rotary(x, x, v, dual(v), pos, cfg),
                     lambda: student.grad_norm([g, dual(g)]), lambda: student.clip_gradients([dual(g)], 1.0),
                     lambda: student.clip_grad_norm_([p], 1.0)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


def _graph_ops(graph):
    return [str(n.target).split(".")[1] for n in graph.graph.nodes if "orda_b200" in str(n.target)]


@pytest.mark.parametrize("pre_dispatch", [False, True])
def test_recorded_calls_are_custom_ops_of_the_graph(pre_dispatch):
    """make_fx sees what passes through the dispatcher only: a call around it would be a constant of the graph."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    with FakeTensorMode():
        x, w = torch.empty(3, 16, device="cuda"), torch.empty(24, 16, device="cuda")
        q, k, v = (torch.empty(*s, device="cuda") for s in ((3, 2, 8), (3, 1, 8), (8,)))
        pos = torch.empty(3, device="cuda", dtype=torch.long)
    cfg = student.RotaryConfig(8)

    def step(x, w, q, k, v, pos):
        q, k = student.qk_norm_rotary(q, k, v, v, pos, cfg)
        return student.gated_linear_unit(x, w, w), *student.rotary_embedding(q, k, pos, cfg)

    graph = make_fx(step, pre_dispatch=pre_dispatch)(x, w, q, k, v, pos)
    assert _graph_ops(graph) == ["rotary", "glu_forward", "rotary"]
    for call in (lambda x: student.grad_norm([x]), lambda x: student.clip_gradients([x], 1.0)):
        with pytest.raises(RuntimeError, match="recorded into a graph"):
            make_fx(call, pre_dispatch=pre_dispatch)(x)
    with pytest.raises(RuntimeError, match="recorded into a graph"):
        torch.jit.trace(lambda x: student.grad_norm([x]), (torch.ones(3),), check_trace=False)


def test_recorded_calls_have_the_shapes_of_plain_ones():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x, w = (torch.empty(*s, device="cuda", dtype=torch.bfloat16) for s in ((2, 3, 16), (24, 16)))
        assert student.gated_linear_unit(x, w, w).shape == (2, 3, 24)
        with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
            student.gated_linear_unit(x.double(), w.double(), w.double())
        with pytest.raises(ValueError, match="activation"):
            student.gated_linear_unit(x, w, w, activation="tanh")


def test_compiled_block_refuses_types_as_the_plain_one_does():
    x, w = torch.randn(4, 16, dtype=torch.float64), torch.randn(24, 16, dtype=torch.float64)
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        torch.compile(lambda x: student.gated_linear_unit(x, w, w), backend="eager")(x)


# ------------------------------------------------------------------------------------------ YaRN's two ramps
def _yarn(**kw):
    return student.RotaryConfig(128, scaling="yarn", factor=8.0, original_positions=4096, **kw).frequencies()


def test_yarn_ramp_in_the_pair_index():
    """128 elements, base 10^4, 4096 positions: a pair turns 4096 / (2 pi) 10^(-i / 16) times, 32 times at
    i = 20.9 and once at i = 45.0; the ramp runs from pair 20 to pair 46."""
    own = student.RotaryConfig(128).frequencies()
    got = _yarn(ramp="index")
    for i, (f, y) in enumerate(zip(own, got)):
        keep = min(1.0, max(0.0, 1.0 - (i - 20) / 26))
        assert y == pytest.approx(f * (keep + (1.0 - keep) / 8), rel=1e-14), i
    assert got[33] == pytest.approx(own[33] * 9 / 16, rel=1e-14)
    turns = _yarn()  # the default: linear in a pair's turns
    assert turns == _yarn(ramp="turns")
    assert min(t / y for t, y in zip(turns, got)) == pytest.approx(0.434, abs=1e-3)
    t33 = 4096 * own[33] / 6.283185307179586
    assert turns[33] == pytest.approx(own[33] * (1 / 8 + 7 / 8 * (t33 - 1) / 31), rel=1e-12)


def test_yarn_ramp_at_its_ends():
    many = student.RotaryConfig(16, scaling="yarn", factor=4.0, original_positions=10 ** 9, ramp="index")
    assert many.frequencies() == student.RotaryConfig(16).frequencies()  # every pair turns often
    few = student.RotaryConfig(16, scaling="yarn", factor=4.0, original_positions=2, ramp="index")
    assert few.frequencies() == pytest.approx([f / 4 for f in student.RotaryConfig(16).frequencies()])
    with pytest.raises(ValueError, match="ramp"):
        student.RotaryConfig(16, ramp="pairs")
    for kw in (dict(base=1.0), dict(base=0.5), dict(beta_slow=0.0)):
        with pytest.raises(ValueError, match="ramp='index'"):
            student.RotaryConfig(16, scaling="yarn", factor=4.0, ramp="index", **kw)


def test_ramp_reaches_the_custom_op():
    c = student.RotaryConfig(64, scaling="yarn", factor=8.0, ramp="index")
    assert student._config_from(*student._config_values(c)) == student.RotaryConfig(
        64, 64, scaling="yarn", factor=8.0, ramp="index", magnitude=c.value_scale)


# ------------------------------------------------------------------------------------------ the training benchmark's model
def test_benchmark_model_without_operators_takes_heads_that_they_refuse():
    from orda_ce_kernel.benchmarks import train_step

    cfg = dict(dim=520, q_heads=1, kv_heads=1, n_layers=1, ffn_dim=16)  # heads of more than 512 elements
    ids = torch.randint(0, 11, (1, 3))
    assert train_step.TinyLM(11, cfg, 4).hidden(ids).shape == (1, 3, 520)
    with pytest.raises(ValueError, match="head_dim"):
        train_step.TinyLM(11, cfg, 4, ops=True)


# ------------------------------------------------------------------------------------------ build
def _build_module():
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "orda-knowledge-distillation-kernel_b200", "build.py")
    spec = importlib.util.spec_from_file_location("orda_build", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("torch_installed", [True, False])
def test_the_library_builds_without_torch(torch_installed, tmp_path, monkeypatch):
    """The commands of a build, recorded instead of run: the binding is compiled where torch is installed only."""
    import os

    b, commands = _build_module(), []

    def run(cmd, check=False):
        commands.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()

    class Popen:
        def __init__(self, cmd):
            run(cmd)

        def wait(self):
            return 0

    monkeypatch.setattr(b, "has_torch", lambda: torch_installed)
    monkeypatch.setattr(b, "_nvcc", lambda: "nvcc")
    monkeypatch.setattr(b, "_binding_flags", lambda: (["-O2"], ["-ltorch"]))
    monkeypatch.setattr(b, "LIB", str(tmp_path / b.LIB_NAME))
    monkeypatch.setattr(b, "BINDING", str(tmp_path / "_student.so"))
    monkeypatch.setattr(b.subprocess, "run", run)
    monkeypatch.setattr(b.subprocess, "Popen", Popen)
    assert b.needs_build()
    b.build()
    assert not b.needs_build()
    assert sorted(os.listdir(tmp_path)) == (["_student.so"] if torch_installed else []) + [b.LIB_NAME]
    assert any(c[0] == "g++" for c in commands) == torch_installed


def test_a_binding_that_does_not_load_names_a_command_that_rebuilds_it(monkeypatch):
    import sys

    monkeypatch.setattr(student, "_binding", None)
    monkeypatch.setitem(sys.modules, "orda_ce_kernel._student", None)  # an import of it fails
    monkeypatch.delattr(sys.modules["orda_ce_kernel"], "_student", raising=False)
    with pytest.raises(RuntimeError, match=r"build.py --force"):
        student.gated_linear_unit(torch.ones(1, 8), torch.ones(8, 8), torch.ones(8, 8))
