"""``orda_ce_kernel.student`` without a GPU: argument errors, the absence of a CPU fallback, the rotary
frequencies, the struct mirrors, the C entry points' own checks, and the custom ops' fake shapes."""
from __future__ import annotations

import ctypes
import math
import os
import shutil
import subprocess

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from orda_ce_kernel import _native, student

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


# ------------------------------------------------------------------------------------------ refusals
def test_no_cpu_fallback():
    x, w = torch.randn(4, 8), torch.randn(16, 8)
    q, k, pos = torch.randn(4, 2, 8), torch.randn(4, 1, 8), torch.arange(4)
    cfg = student.RotaryConfig(8)
    for call in (lambda: student.gated_linear_unit(x, w, w), lambda: student.rotary_embedding(q, k, pos, cfg),
                 lambda: student.qk_norm_rotary(q, k, torch.ones(8), torch.ones(8), pos, cfg),
                 lambda: student.grad_norm([x]), lambda: student.clip_gradients([x], 1.0)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


@pytest.mark.parametrize("change,match", [
    (dict(activation="tanh"), "activation must be"),
    (dict(up=torch.randn(15, 8)), "one shape"),
    (dict(gate=torch.randn(16), up=torch.randn(16)), "one shape"),
    (dict(x=torch.randn(4, 9)), "x must have shape"),
    (dict(x=torch.randn(4, 8, dtype=torch.float64)), "float32, float16 or bfloat16"),
    (dict(gate=torch.randn(0, 8), up=torch.randn(0, 8)), "must not be empty"),
])
def test_gated_linear_unit_refuses(change, match):
    a = dict(x=torch.randn(4, 8), gate=torch.randn(16, 8), up=torch.randn(16, 8), activation="silu") | change
    with pytest.raises(ValueError, match=match):
        student.gated_linear_unit(a["x"], a["gate"], a["up"], activation=a["activation"])


@pytest.mark.parametrize("change,error,match", [
    (dict(config=None), TypeError, "RotaryConfig"),
    (dict(q=torch.randn(4, 8)), ValueError, "tokens, heads, head_dim"),
    (dict(k=torch.randn(5, 1, 8)), ValueError, "same tokens"),
    (dict(k=torch.randn(4, 1, 6)), ValueError, "head_dim=8"),
    (dict(k=torch.randn(4, 1, 8).half()), ValueError, "must both be"),
    (dict(pos=torch.arange(4).float()), ValueError, "int32 or int64"),
    (dict(pos=torch.arange(3)), ValueError, "positions must have shape"),
])
def test_rotary_refuses(change, error, match):
    a = dict(q=torch.randn(4, 2, 8), k=torch.randn(4, 1, 8), pos=torch.arange(4), config=student.RotaryConfig(8)) | change
    with pytest.raises(error, match=match):
        student.rotary_embedding(a["q"], a["k"], a["pos"], a["config"])
    with pytest.raises(error, match=match):
        student.qk_norm_rotary(a["q"], a["k"], torch.ones(8), torch.ones(8), a["pos"], a["config"])


def test_qk_norm_refuses_weights_and_eps():
    q, k, pos, cfg = torch.randn(4, 2, 8), torch.randn(4, 1, 8), torch.arange(4), student.RotaryConfig(8)
    one = torch.ones(8)
    for wq, wk, eps, match in ((torch.ones(7), one, 1e-6, "q_weight must have shape"),
                               (one, torch.ones(8, 1), 1e-6, "k_weight must have shape"),
                               (one, one.half(), 1e-6, "one dtype")):
        with pytest.raises(ValueError, match=match):
            student.qk_norm_rotary(q, k, wq, wk, pos, cfg, eps)
    for eps in (-1e-6, math.nan):
        with pytest.raises(ValueError, match="eps"):
            student.qk_norm_rotary(q, k, one, one, pos, cfg, eps)


@pytest.mark.parametrize("kw,match", [
    (dict(head_dim=0), "head_dim"), (dict(head_dim=514), "head_dim"), (dict(head_dim=9), "rotary_dim"),
    (dict(head_dim=8, rotary_dim=10), "rotary_dim"), (dict(head_dim=8, rotary_dim=0), "rotary_dim"),
    (dict(head_dim=8, layout="both"), "layout"), (dict(head_dim=8, scaling="log"), "scaling"),
    (dict(head_dim=8, base=0.0), "base"), (dict(head_dim=8, factor=0.5), "factor"),
    (dict(head_dim=8, rotary_dim=2, scaling="ntk", factor=2.0), "ntk"),
    (dict(head_dim=8, scaling="yarn", factor=2.0, beta_fast=1.0), "yarn"),
])
def test_rotary_config_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        student.RotaryConfig(**kw)


@pytest.mark.parametrize("max_norm,eps", [(-1.0, 1e-6), (math.nan, 1e-6), (1.0, -1.0)])
def test_clip_refuses_limits(max_norm, eps):
    with pytest.raises(ValueError):
        student.clip_gradients([torch.ones(3)], max_norm, eps=eps)
    p = torch.nn.Parameter(torch.ones(3))
    p.grad = torch.ones(3)
    with pytest.raises(ValueError):
        student.clip_grad_norm_([p], max_norm, eps=eps)


def test_clip_refuses_types_and_accepts_nothing():
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        student.grad_norm([torch.ones(3, dtype=torch.float64)])
    with pytest.raises(ValueError, match="strided"):
        student.grad_norm([torch.ones(3).to_sparse()])
    assert float(student.grad_norm([])) == 0.0
    clipped, norm = student.clip_gradients([], 1.0)
    assert clipped == [] and float(norm) == 0.0
    assert float(student.clip_grad_norm_([torch.nn.Parameter(torch.ones(2))], 1.0)) == 0.0


# ------------------------------------------------------------------------------------------ frequencies
def test_frequencies_follow_their_formulas():
    plain = student.RotaryConfig(16, rotary_dim=8, base=100.0).frequencies()
    assert plain == pytest.approx([100.0 ** (-i / 4) for i in range(4)], rel=1e-15)
    lin = student.RotaryConfig(16, rotary_dim=8, base=100.0, scaling="linear", factor=4.0)
    assert lin.frequencies() == pytest.approx([f / 4 for f in plain], rel=1e-15) and lin.value_scale == 1.0
    ntk = student.RotaryConfig(16, rotary_dim=8, base=100.0, scaling="ntk", factor=4.0).frequencies()
    # the slowest pair is stretched by the whole factor, the fastest not at all
    assert ntk[0] == 1.0 and ntk[-1] == pytest.approx(plain[-1] / 4, rel=1e-12)
    yarn = student.RotaryConfig(64, scaling="yarn", factor=8.0, original_positions=4096)
    base = student.RotaryConfig(64).frequencies()
    for y, f in zip(yarn.frequencies(), base):
        turns = 4096 * f / (2 * math.pi)
        if turns >= 32:
            assert y == pytest.approx(f, rel=1e-15)
        elif turns <= 1:
            assert y == pytest.approx(f / 8, rel=1e-15)
        else:
            assert f / 8 < y < f
    assert yarn.value_scale == pytest.approx(0.1 * math.log(8.0) + 1.0)
    assert student.RotaryConfig(64, scaling="yarn", factor=8.0, magnitude=1.0).value_scale == 1.0


def test_config_survives_its_plain_values():
    for c in (student.RotaryConfig(96, 32, 5e5, "interleaved", "yarn", 16.0, 8192, 20.0, 2.0),
              student.RotaryConfig(64), student.RotaryConfig(64, scaling="ntk", factor=2.0)):
        back = student._config_from(*student._config_values(c))
        assert back.frequencies() == c.frequencies() and back.value_scale == c.value_scale
        assert (back.layout, back.dim, back.head_dim) == (c.layout, c.dim, c.head_dim)


def test_config_copies_and_pickles():
    import copy
    import pickle

    c = student.RotaryConfig(64, scaling="yarn", factor=2.0)
    student._plan(c)
    for d in (copy.deepcopy(c), pickle.loads(pickle.dumps(c)), copy.copy(c)):
        assert d == c and hash(d) == hash(c) and d.frequencies() == c.frequencies()
        student._plan(d)


def test_training_benchmark_model_without_operators_runs_on_cpu():
    from orda_ce_kernel.benchmarks import train_step

    cfg = dict(dim=32, q_heads=4, kv_heads=2, n_layers=1, ffn_dim=64)
    ids = torch.randint(0, 97, (2, 8))
    lm = train_step.TinyLM(97, cfg, 8, qk_norm=True)
    lm.hidden(ids).sum().backward()
    assert lm.blocks[0].attn.q_norm.scale.grad is not None
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        train_step.TinyLM(97, cfg, 8, ops=True).hidden(ids)


# ------------------------------------------------------------------------------------------ C boundary
@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc")
def test_struct_mirrors_match_the_header(tmp_path):
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "orda_b200_student.h"\nint main(void) {'
                   'printf("%zu %zu %zu %zu %zu", sizeof(orda_glu_args_t), sizeof(orda_rotary_args_t),'
                   'sizeof(orda_tensor_list_t), offsetof(orda_glu_args_t, device_status),'
                   'offsetof(orda_rotary_args_t, dweight)); return 0; }')
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)],
                   check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(_native.GluArgs), ctypes.sizeof(_native.RotaryArgs), ctypes.sizeof(_native.TensorList),
                   _native.GluArgs.device_status.offset, _native.RotaryArgs.dweight.offset]


def _glu(**kw):
    a = dict(abi_version=_native.ABI_VERSION, dtype=_native.BF16, activation=0, rows=4, hidden=16, ffn=8, x=16, ld_x=16,
             gate=16, ld_gate=16, up=16, ld_up=16, h=16, ld_h=8, ld_pre=8, device_status=16) | kw
    return _native.GluArgs(**a)


@pytest.mark.parametrize("kw,code", [
    (dict(abi_version=9), _native.ERR_INVALID_ARGUMENT), (dict(dtype=5), _native.ERR_INVALID_ARGUMENT),
    (dict(activation=4), _native.ERR_INVALID_ARGUMENT), (dict(rows=-1), _native.ERR_INVALID_ARGUMENT),
    (dict(hidden=0), _native.ERR_INVALID_ARGUMENT), (dict(x=None), _native.ERR_INVALID_ARGUMENT),
    (dict(h=None), _native.ERR_INVALID_ARGUMENT), (dict(rows=129, device_status=None), _native.ERR_INVALID_ARGUMENT), (dict(pre_gate=16), _native.ERR_INVALID_ARGUMENT),
    (dict(ld_gate=8), _native.ERR_INVALID_ARGUMENT), (dict(x=24), _native.ERR_ALIGNMENT),
    (dict(hidden=12), _native.ERR_ALIGNMENT), (dict(ld_up=20), _native.ERR_ALIGNMENT),
    (dict(rows=1 << 31), _native.ERR_UNSUPPORTED), (dict(rows=0), _native.OK),
])
def test_c_glu_checks(kw, code):
    assert _native.load().orda_glu_forward(_glu(**kw), None) == code


def test_c_glu_backward_checks():
    lib = _native.load()
    ok = dict(pre_gate=16, pre_up=16, dh=16, dx=16, dweights=16, h=None, grad_cols=16)
    size = lib.orda_glu_backward_workspace_bytes(_glu(**ok))
    assert size >= 4 * 16 * 2
    assert lib.orda_glu_backward(_glu(**ok), 256, size - 1, None) == _native.ERR_WORKSPACE
    assert lib.orda_glu_backward(_glu(**ok), None, size, None) == _native.ERR_WORKSPACE
    assert lib.orda_glu_backward(_glu(**ok | dict(dh=None)), 256, size, None) == _native.ERR_INVALID_ARGUMENT
    assert lib.orda_glu_backward(_glu(**ok | dict(dx=8)), 256, size, None) == _native.ERR_ALIGNMENT
    for cols in (0, 17):
        assert lib.orda_glu_backward(_glu(**ok | dict(grad_cols=cols)), 256, size, None) == _native.ERR_INVALID_ARGUMENT


def test_c_pointers_inside_an_element_are_refused():
    lib = _native.load()
    assert lib.orda_glu_forward(_glu(h=17), None) == _native.ERR_ALIGNMENT
    assert lib.orda_glu_forward(_glu(dtype=_native.F32, pre_gate=16, pre_up=16, h=18), None) == _native.ERR_ALIGNMENT
    assert lib.orda_glu_backward(_glu(pre_gate=16, pre_up=16, dh=17, dx=16, grad_cols=16), 256, 1 << 20,
                                 None) == _native.ERR_ALIGNMENT
    for kw in (dict(x=(16, 17)), dict(out=(17, 16)), dict(positions=18), dict(positions=20, positions_int64=1),
               dict(weight=(16, 18), weight_dtype=_native.F32)):
        a, _f = _rot(**kw)
        assert lib.orda_rotary_forward(a, None) == _native.ERR_ALIGNMENT, kw
    full = dict(weight=(16, 16), dweight=(16, 16), dy=(16, 16), weight_dtype=_native.F32)
    size = lib.orda_qk_norm_rotary_backward_workspace_bytes(_rot(**full)[0])
    for kw, workspace in ((dict(dy=(17, 16)), 256), (dict(dweight=(16, 18)), 256), ({}, 264)):
        a, _f = _rot(**full | kw)
        assert lib.orda_qk_norm_rotary_backward(a, workspace, size, None) == _native.ERR_ALIGNMENT, kw
    one = _list([16], [4], [0])
    size = lib.orda_clip_workspace_bytes(one)
    assert lib.orda_clip_gradients(one, 1.0, 1e-6, 16, 264, size, None) == _native.ERR_ALIGNMENT
    assert lib.orda_clip_gradients(one, 1.0, 1e-6, 18, 256, size, None) == _native.ERR_ALIGNMENT


def test_c_pad_rows_checks():
    def call(count=1, src=(16,), ld=(3,), rows=(4,), cols=3, dst=(16,)):
        n = len(src)
        return _native.load().orda_pad_rows(count, (ctypes.c_void_p * n)(*src), (ctypes.c_int64 * n)(*ld),
                                            (ctypes.c_int64 * n)(*rows), cols, (ctypes.c_void_p * n)(*dst), None)

    assert call(count=4) == call(cols=0) == call(rows=(-1,)) == call(src=(None,)) == _native.ERR_INVALID_ARGUMENT
    assert call(src=(17,)) == call(dst=(24,)) == _native.ERR_ALIGNMENT
    assert call(rows=(0,)) == call(count=0) == _native.OK


def _rot(**kw):
    f = (ctypes.c_uint64 * 4)(1, 2, 3, 4)
    a = dict(abi_version=_native.ABI_VERSION, dtype=_native.BF16, batch=1, seq=2, heads=(2, 1), head_dim=8, rotary_dim=8,
             layout=0, x=(16, 16), out=(16, 16), positions=16, turns=ctypes.addressof(f), magnitude=1.0) | kw
    return _native.RotaryArgs(**a), f


@pytest.mark.parametrize("kw,code", [
    (dict(abi_version=9), _native.ERR_INVALID_ARGUMENT), (dict(rotary_dim=7), _native.ERR_INVALID_ARGUMENT),
    (dict(rotary_dim=10), _native.ERR_INVALID_ARGUMENT), (dict(layout=2), _native.ERR_INVALID_ARGUMENT),
    (dict(head_dim=1024, rotary_dim=8), _native.ERR_UNSUPPORTED), (dict(positions=None), _native.ERR_INVALID_ARGUMENT),
    (dict(turns=None), _native.ERR_INVALID_ARGUMENT), (dict(x=(16, None)), _native.ERR_INVALID_ARGUMENT),
    (dict(weight=(16, None)), _native.ERR_INVALID_ARGUMENT), (dict(batch=1 << 20, seq=1 << 20), _native.ERR_UNSUPPORTED),
    (dict(batch=0), _native.OK), (dict(heads=(0, 0)), _native.OK),
])
def test_c_rotary_checks(kw, code):
    a, _f = _rot(**kw)
    assert _native.load().orda_rotary_forward(a, None) == code


def test_c_rotary_turns():
    lib = _native.load()
    angles = [0.0, 1.0, 2 * math.pi * 0.25, -1.0, 1e-18, -1e-30, 2.5e9]
    out = (ctypes.c_uint64 * len(angles))()
    assert lib.orda_rotary_turns((ctypes.c_double * len(angles))(*angles), len(angles), out) == _native.OK
    for a, t in zip(angles, out):
        off = (t / 2.0 ** 64 - a / (2 * math.pi)) % 1.0
        assert min(off, 1.0 - off) <= 2.0 ** -53 * (1 + abs(a)), a
    for bad in (math.inf, math.nan):
        assert lib.orda_rotary_turns((ctypes.c_double * 1)(bad), 1, out) == _native.ERR_INVALID_ARGUMENT
    assert lib.orda_rotary_turns(None, 1, out) == _native.ERR_INVALID_ARGUMENT


def test_c_norm_backward_checks():
    lib = _native.load()
    full = dict(weight=(16, 16), dweight=(16, 16), dy=(16, 16), weight_dtype=_native.F32)
    a, _f = _rot(**full)
    size = lib.orda_qk_norm_rotary_backward_workspace_bytes(a)
    assert size > 0
    assert lib.orda_qk_norm_rotary_backward(a, 256, size - 1, None) == _native.ERR_WORKSPACE
    for lost in ("weight", "dweight", "dy"):
        b, _g = _rot(**{k: v for k, v in full.items() if k != lost})
        assert lib.orda_qk_norm_rotary_backward(b, 256, size, None) == _native.ERR_INVALID_ARGUMENT


def _list(addresses, numel, dtypes, dst=None):
    n = len(addresses)
    return _native.TensorList(_native.ABI_VERSION, n, (ctypes.c_void_p * n)(*addresses),
                              None if dst is None else (ctypes.c_void_p * n)(*dst), (ctypes.c_int64 * n)(*numel),
                              (ctypes.c_int32 * n)(*dtypes))


def test_c_clip_checks():
    lib = _native.load()
    good = _list([16, 32], [4, 4], [0, 2])
    size = lib.orda_clip_workspace_bytes(good)
    assert size > 0
    call = lib.orda_clip_gradients
    assert call(good, 1.0, 1e-6, None, 256, size, None) == _native.ERR_INVALID_ARGUMENT
    assert call(good, -1.0, 1e-6, 16, 256, size, None) == _native.ERR_INVALID_ARGUMENT
    assert call(good, math.nan, 1e-6, 16, 256, size, None) == _native.ERR_INVALID_ARGUMENT
    assert call(good, 1.0, 1e-6, 16, 256, size - 1, None) == _native.ERR_WORKSPACE
    assert call(_list([16], [-1], [0]), 1.0, 1e-6, 16, 256, size, None) == _native.ERR_INVALID_ARGUMENT
    assert call(_list([16], [4], [3]), 1.0, 1e-6, 16, 256, size, None) == _native.ERR_INVALID_ARGUMENT
    assert call(_list([None], [4], [0]), 1.0, 1e-6, 16, 256, size, None) == _native.ERR_INVALID_ARGUMENT
    assert call(_list([18], [4], [0]), 1.0, 1e-6, 16, 256, size, None) == _native.ERR_ALIGNMENT
    assert call(_list([16], [4], [2], dst=[33]), 1.0, 1e-6, 16, 256, size, None) == _native.ERR_ALIGNMENT
    many = _list([16] * 2000, [4] * 2000, [0] * 2000)
    assert lib.orda_clip_workspace_bytes(many) > size


# ------------------------------------------------------------------------------------------ torch.compile
def test_fake_shapes():
    with FakeTensorMode():
        x, w = torch.empty(6, 16, dtype=torch.bfloat16), torch.empty(13, 16, dtype=torch.bfloat16)
        h, pre = torch.ops.orda_b200.glu_forward(x, w, w, 0)
        assert h.shape == (6, 13) and pre.shape == (2, 6, 16) and h.dtype == torch.bfloat16
        dx, dg, du = torch.ops.orda_b200.glu_backward(h, x, w, w, pre, 0)
        assert dx.shape == x.shape and dg.shape == du.shape == w.shape
        q, k, pos = torch.empty(2, 5, 4, 32), torch.empty(2, 5, 2, 32), torch.empty(2, 5, dtype=torch.long)
        cfg = student._config_values(student.RotaryConfig(32))
        oq, ok_ = torch.ops.orda_b200.rotary(q, k, pos, None, None, 0.0, False, *cfg)
        assert oq.shape == q.shape and ok_.shape == k.shape
        wq = torch.empty(32)
        gs = torch.ops.orda_b200.qk_norm_rotary_backward(oq, ok_, q, k, pos, wq, wq, 1e-6, *cfg)
        assert [t.shape for t in gs] == [q.shape, k.shape, wq.shape, wq.shape]


def test_public_calls_trace_without_graph_break():
    class Step(torch.nn.Module):
        def forward(self, x, gate, up, q, k, wq, wk, pos):
            h = student.gated_linear_unit(x, gate, up, activation="gelu")
            cfg = student.RotaryConfig(32, layout="interleaved")
            q, k = student.qk_norm_rotary(q, k, wq, wk, pos, cfg)
            return h, *student.rotary_embedding(q, k, pos, cfg)

    with FakeTensorMode(allow_non_fake_inputs=True):
        def cuda(*shape, dtype=torch.bfloat16, grad=True):
            return torch.empty(*shape, device="cuda", dtype=dtype, requires_grad=grad)

        args = (cuda(2, 5, 16), cuda(24, 16), cuda(24, 16), cuda(2, 5, 4, 32), cuda(2, 5, 2, 32), cuda(32), cuda(32),
                cuda(5, dtype=torch.long, grad=False))
    ep = torch.export.export(Step(), args, strict=True)
    names = [str(n.target) for n in ep.graph.nodes if n.op == "call_function" and "orda_b200" in str(n.target)]
    assert [n.split(".")[1] for n in names] == ["glu_forward", "rotary", "rotary"]
