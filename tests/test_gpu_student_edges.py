"""GPU tests of ``orda_ce_kernel.student`` at the edges of values, sizes and ways of calling.

Tolerances as in ``test_gpu_student``: worked out per element, ``half`` is one rounding.
"""
from __future__ import annotations

import math

import pytest
import torch

from orda_ce_kernel import _native, student
from test_gpu_student import BF16, FP16, FP32, check_rotary, glu64, glu_inputs, half, randn, within

pytestmark = pytest.mark.gpu

ACTS = ["silu", "gelu", "gelu_tanh", "relu"]
ACT = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu,
       "gelu_tanh": lambda g: torch.nn.functional.gelu(g, approximate="tanh")}


def glu_pass(x, wg, wu, act, dh):
    """(h, dx, dgate, dup)"""
    leaves = [t.detach().requires_grad_(True) for t in (x, wg, wu)]
    h = student.gated_linear_unit(*leaves, activation=act)
    return (h.detach(), *torch.autograd.grad(h, leaves, dh))


# ------------------------------------------------------------------------------------------ values that are not finite
# rows: each 16-bit forward kernel (streamed weights, weights first, pair GEMM); fp32
@pytest.mark.parametrize("n", [5, 40, 300])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("act", ACTS)
def test_glu_gate_weight_that_is_not_finite_shows(act, dtype, n):
    """A NaN in one gate row reaches its feature of h and every gradient that reads it, and nothing else;
    infinite products give what the formula gives."""
    x, wg, wu, dh = glu_inputs(n, 64, 72, dtype, 11)
    clean = glu_pass(x, wg, wu, act, dh)
    others = torch.arange(72, device="cuda") != 7
    bad = wg.clone()
    bad[7, 5] = math.nan
    h, dx, dgate, dup = glu_pass(x, bad, wu, act, dh)
    for row in (h[:, 7], dx, dgate[7], dup[7]):
        assert torch.isnan(row).all()
    assert torch.equal(h[:, others], clean[0][:, others])
    assert torch.equal(dgate[others], clean[2][others]) and torch.equal(dup[others], clean[3][others])
    bad[7, 5] = math.inf
    h = glu_pass(x, bad, wu, act, dh)[0]
    want = ACT[act](x.double() @ bad.double().T) * (x.double() @ wu.double().T)
    assert torch.equal(h[:, others], clean[0][:, others])
    assert torch.equal(torch.isnan(h[:, 7]), torch.isnan(want[:, 7]))
    keep = ~torch.isnan(want[:, 7])
    assert bool(keep.any()) and torch.equal(h[keep, 7].double(), want[keep, 7])  # infinities, and zeros of relu


@pytest.mark.parametrize("n", [5, 40, 300])
@pytest.mark.parametrize("act", ACTS)
def test_glu_fp16_products_behind_the_types_range(act, n):
    """Gate products of about +-1e5 beside small and large up products: h is formed from fp32 products, and the
    gradients have to be finite wherever the formula's are."""
    x, wg, wu, dh = glu_inputs(n, 64, 75, FP16, 21)
    x, dh = x * 30, (dh * 2e-4).to(FP16)
    wg, wu = wg / 30, wu / 30
    wg[:4] *= 1e5  # |x| |w| is about 240 / sqrt(64) / 30 = 1 without these
    wu[2:6] *= 1e5
    g, u = x.double() @ wg.double().T, x.double() @ wu.double().T
    assert bool((g < -65520).any()) and bool((g > 65520).any()) and bool((u.abs() > 65520).any())
    want = glu64(x, wg, wu, act, dh)
    h, *grads = glu_pass(x, wg, wu, act, dh)
    fits = want["h"][0].abs() < 65000
    within(h[fits], want["h"][0][fits], want["h"][1][fits], "h")
    for name, got in zip(("dx", "dgate", "dup"), grads):
        assert float(want[name][0].abs().max()) < 60000
        within(got, *want[name], name)


# ------------------------------------------------------------------------------------------ clipping in place
def _params(*grads):
    params = [torch.nn.Parameter(torch.empty(g.shape, device="cuda", dtype=g.dtype)) for g in grads]
    for p, g in zip(params, grads):
        p.grad = g
    return params


def test_clip_refusals_leave_every_gradient_as_it_was():
    flat = torch.ones(100, device="cuda")
    first = torch.ones(3, device="cuda")
    for bad in (flat[10:20], torch.ones(1, 8, device="cuda").expand(4, 8)):
        with pytest.raises(ValueError):
            student.clip_grad_norm_(_params(first, flat, bad), 1e-3)
        assert bool((flat == 1).all()) and bool((first == 1).all()) and bool((bad == 1).all())


def test_clip_gradients_between_each_other():
    flat = randn(101, seed=3)
    before = flat.double()
    norm = student.clip_grad_norm_(_params(flat[::2], flat[1::2]), 1.0)
    want = float(before.square().sum().sqrt())
    assert float(norm) == pytest.approx(want, rel=2.0 ** -23)
    # the factor, its product and the value are rounded to fp32
    within(flat, before / (want + 1e-6), before.abs() / want * 2.0 ** -22)


# ------------------------------------------------------------------------------------------ exact sums
def integers(*shape, seed, dtype, density):
    """-1, 0 and 1; `density` of them not 0."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    u = torch.rand(shape, generator=g, device="cuda")
    return (u < density / 2).to(dtype) - (u > 1 - density / 2).to(dtype)


def check_exact(x, wg, wu, dh):
    """ReLU block on small integers. Products of at most 256 are exact in every type, and so are dg and du; all
    sums are integers below 2^24, exact in fp32 in any order. Each result is the exact one, rounded once."""
    dt = x.dtype
    got = glu_pass(x, wg, wu, "relu", dh)
    x, wg, wu, dh = (t.double() for t in (x, wg, wu, dh))
    g, u = x @ wg.T, x @ wu.T
    assert float(g.abs().max()) <= 256 and float(u.abs().max()) <= 256
    a, d = g.relu(), (g > 0).double()
    dg, du = dh * u * d, dh * a
    for name, y, want in zip(("h", "dx", "dgate", "dup"), got, (a * u, dg @ wg + du @ wu, dg.T @ x, du.T @ x)):
        assert float(want.abs().max()) < 2 ** 24
        wrong = y != want.to(dt)
        assert not bool(wrong.any()), (name, wrong.nonzero()[:3].tolist(), int(wrong.sum()))


@pytest.mark.parametrize("n,h,f", [(65535 * 64 + 1, 8, 3), (2, 3, 65535 * 32 + 40)])
def test_glu_fp32_sizes_of_more_than_65535_tiles(n, h, f):
    """Rows (h, dx), and features (weight gradients), behind 65535 tiles of 64."""
    check_exact(integers(n, h, seed=1, dtype=FP32, density=0.7), integers(f, h, seed=2, dtype=FP32, density=0.7),
                integers(f, h, seed=3, dtype=FP32, density=0.7), integers(n, f, seed=4, dtype=FP32, density=0.1))


# ------------------------------------------------------------------------------------------ errors of a launch
def test_a_failed_launch_is_reported_once():
    lib, stream = _native.load(), torch.cuda.current_stream().cuda_stream
    g, q = [torch.ones(4, device="cuda")], randn(3, 2, 16, seed=1)
    pos, cfg = torch.arange(3, device="cuda"), student.RotaryConfig(16)
    calls = (lambda: student.grad_norm(g), lambda: student.rotary_embedding(q, q, pos, cfg)[0],
             lambda: glu_pass(*glu_inputs(40, 64, 72, BF16, 3)[:3], "silu", torch.ones(40, 72, device="cuda", dtype=BF16))[1],
             lambda: glu_pass(*glu_inputs(300, 64, 72, BF16, 3)[:3], "silu", torch.ones(300, 72, device="cuda", dtype=BF16))[1])
    want = [c() for c in calls]
    for call, w in zip(calls, want):
        assert lib.orda_debug_failed_launch(stream) == _native.ERR_CUDA
        assert torch.equal(call(), w)


# one product each, K-split products, rows of a multiple of 8 and not (grad_cols)
@pytest.mark.parametrize("n,h,cols,f", [(300, 64, 64, 75), (2048, 1024, 1024, 2816), (1111, 1000, 997, 2730)])
def test_c_glu_results_marked_by_a_timeout(n, h, cols, f):
    """The marks of a wait that timed out make the first value of h, of dx and of each weight's gradient NaN,
    whether the gradients come from one product or from partial sums, and nothing else."""
    x, wg, wu, dh = glu_inputs(n, h, f, BF16, 61)
    lib, fp = _native.load(), (f + 7) // 8 * 8
    stream = torch.cuda.current_stream().cuda_stream

    def run(forward, backward):
        y, pre = torch.empty(n, f, device="cuda", dtype=BF16), torch.empty(2, n, fp, device="cuda", dtype=BF16)
        dx, dw = torch.empty(n, cols, device="cuda", dtype=BF16), torch.zeros(fp + f, cols, device="cuda", dtype=BF16)
        status = torch.zeros(1, device="cuda", dtype=torch.int32)
        a = _native.GluArgs(abi_version=_native.ABI_VERSION, dtype=_native.BF16, activation=_native.ACT_SILU, rows=n, hidden=h,
                            ffn=f, x=x.data_ptr(), ld_x=h, gate=wg.data_ptr(), ld_gate=h, up=wu.data_ptr(), ld_up=h,
                            h=y.data_ptr(), ld_h=f, pre_gate=pre[0].data_ptr(), ld_pre=fp, pre_up=pre[1].data_ptr(),
                            grad_cols=cols, dh=dh.data_ptr(), dx=dx.data_ptr(), dweights=dw.data_ptr(),
                            device_status=status.data_ptr())
        assert forward(a, stream) == _native.OK
        need = lib.orda_glu_backward_workspace_bytes(a)
        ws = torch.empty(need, device="cuda", dtype=torch.uint8)
        assert backward(a, ws.data_ptr(), need, stream) == _native.OK
        return y, dx, dw[:f], dw[fp:]

    want = run(lib.orda_glu_forward, lib.orda_glu_backward)
    got = run(lib.orda_debug_glu_forward_marked, lib.orda_debug_glu_backward_marked)
    for a, b in zip(got, want):
        assert bool(torch.isnan(a[0, 0])) and bool(torch.isfinite(b).all())
        a[0, 0] = b[0, 0]
        assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------ recorders
def _block(x, wg, wu, q, k, wq, wk, pos):
    cfg = student.RotaryConfig(64)
    a, b = student.qk_norm_rotary(q, k, wq, wk, pos, cfg)
    return student.gated_linear_unit(x, wg, wu), *student.rotary_embedding(a, b, pos, cfg)


def _block_inputs(seed):
    x, wg, wu, _ = glu_inputs(40, 64, 72, BF16, seed)
    q, k = randn(40, 2, 64, seed=seed + 4, dtype=BF16), randn(40, 1, 64, seed=seed + 5, dtype=BF16)
    return x, wg, wu, q, k, randn(64, seed=seed + 6), randn(64, seed=seed + 7), torch.arange(40, device="cuda") + seed


@pytest.mark.parametrize("how", ["make_fx", "jit"])
def test_recorded_graphs_compute_from_their_inputs(how):
    from torch.fx.experimental.proxy_tensor import make_fx

    first, second = _block_inputs(1), _block_inputs(50)
    graph = make_fx(_block)(*first) if how == "make_fx" else torch.jit.trace(_block, first)
    for ins in (first, second):
        for a, b in zip(graph(*ins), _block(*ins)):
            assert torch.equal(a, b)


def test_calls_under_a_dispatch_mode_are_seen_and_differentiated():
    from torch.utils._python_dispatch import TorchDispatchMode

    seen = []

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    def run():
        *leaves, pos = _block_inputs(7)
        leaves = [t.requires_grad_(True) for t in leaves]
        out = _block(*leaves, pos)
        grads = torch.autograd.grad(sum(o.float().square().sum() for o in out), leaves)
        clipped, norm = student.clip_gradients(grads, 1.0)
        return [*out, *clipped, norm]

    want = run()
    assert not seen
    with Watch():
        got = run()
    assert sum("orda_b200.glu" in s for s in seen) == 2 and sum("orda_b200.rotary" in s for s in seen) == 3
    for a, b in zip(got, want):
        assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------ lazily negated and zero tensors
def test_tensors_whose_values_are_not_in_memory_as_such():
    """Views that stand for the negatives of what they point at (the imaginary part of a conjugate), and zero
    tensors without memory, as inputs and as gradients."""
    def neg(t):
        return torch._neg_view((-t).clone())

    x, wg, wu, q, k, wq, wk, pos = ins = _block_inputs(3)
    want = _block(*ins)
    for a, b in zip(_block(*(neg(t) for t in ins)), want):
        assert torch.equal(a, b)
    leaves = [t.detach().requires_grad_(True) for t in ins[:-1]]
    dy = [randn(*o.shape, seed=9 + i, dtype=BF16) for i, o in enumerate(want)]
    plain = torch.autograd.grad(_block(*leaves, pos), leaves, dy)
    for a, b in zip(torch.autograd.grad(_block(*leaves, pos), leaves, [neg(d) for d in dy]), plain):
        assert torch.equal(a, b)
    part = torch.conj(torch.complex(q.float(), q.float())).imag[..., :1]  # dense: one element a head
    assert part.is_neg()
    for t in (part, neg(wg), x):
        clipped, norm = student.clip_gradients([t], 1.0)
        assert torch.equal(norm, student.grad_norm([t.clone()]))
        assert torch.equal(clipped[0], student.clip_gradients([t.clone()], 1.0)[0][0])
    g = neg(wg)
    norm = student.clip_grad_norm_(_params(g), 1.0)
    assert torch.equal(g.clone(), student.clip_gradients([wg], 1.0)[0][0])
    zero = torch._efficientzerotensor((40, 64), device="cuda", dtype=BF16)
    assert not student.gated_linear_unit(zero, wg, wu).any() and float(student.grad_norm([zero, wg])) == float(norm)


# ------------------------------------------------------------------------------------------ saved-tensor hooks
def _reversed_strides(t):
    """The same values in memory in the opposite order of dimensions."""
    dims = list(range(t.ndim))[::-1]
    return t.permute(dims).contiguous().permute(dims)


def _behind_a_boundary(t):
    """The same values starting one element behind a 16-byte boundary."""
    return torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape)


@pytest.mark.parametrize("unpack", [_reversed_strides, _behind_a_boundary, lambda t: t.cpu().cuda()])
@pytest.mark.parametrize("n,h", [(40, 64), (300, 66)])
def test_saved_tensors_that_come_back_with_other_strides(unpack, n, h):
    x, wg, wu, dh = glu_inputs(n, h, 75, BF16, 71)
    *_, q, k, wq, wk, pos = _block_inputs(5)
    cfg = student.RotaryConfig(64, rotary_dim=32)
    leaves = [t.detach().requires_grad_(True) for t in (x, wg, wu, q, k, wq, wk)]
    dq, dk = randn(*q.shape, seed=6, dtype=BF16), randn(*k.shape, seed=7, dtype=BF16)

    def run():
        a, b = student.qk_norm_rotary(*leaves[3:], pos, cfg)
        a, b = student.rotary_embedding(a, b, pos, cfg)
        out = (student.gated_linear_unit(*leaves[:3]), a, b)
        return torch.autograd.grad(out, leaves, (dh, dq, dk))

    want = run()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        got = run()
    for a, b in zip(got, want):
        # weight gradients of the norms are added up in another order where heads are read in narrower vectors
        torch.testing.assert_close(a, b, rtol=2 * half(b.dtype) if b.dtype != FP32 else 1e-5, atol=1e-5)


def test_saved_tensors_that_come_back_as_others_are_refused():
    x, wg, wu, dh = glu_inputs(40, 64, 72, BF16, 71)
    *_, q, k, wq, wk, pos = _block_inputs(5)
    for call, leaf in ((lambda t: student.gated_linear_unit(t, wg, wu), x),
                       (lambda t: student.qk_norm_rotary(t, k, wq, wk, pos, student.RotaryConfig(64))[0], q),
                       (lambda t: student.rotary_embedding(t, k, pos, student.RotaryConfig(64))[0], q)):
        for unpack in (lambda t: t.cpu(), lambda t: t[1:], lambda t: t[..., :1]):
            leaf = leaf.detach().requires_grad_(True)
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
                y = call(leaf)
            with pytest.raises((ValueError, RuntimeError)):
                y.sum().backward()


# ------------------------------------------------------------------------------------------ large finite values
@pytest.mark.parametrize("n", [5, 40, 300])
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("act", ACTS)
def test_glu_gates_whose_square_is_infinite(act, dtype, n):
    """Gates of +-1.6e21: activations and derivatives are at their limits (g and 1, or 0), and finite."""
    x = torch.full((n, 16), 1e10, device="cuda", dtype=dtype)
    wg = torch.full((24, 16), 1e10, device="cuda", dtype=dtype)
    wg[::2] *= -1
    wu, dh = torch.full_like(wg, 1e-10), torch.full((n, 24), 1e-20, device="cuda", dtype=dtype)
    got = glu_pass(x, wg, wu, act, dh)
    x, wg, wu, dh = (t.double() for t in (x, wg, wu, dh))
    g, u = x @ wg.T, x @ wu.T
    a, d = g.relu(), (g > 0).double()
    dg, du = dh * u * d, dh * a
    # nothing cancels: the products, dg and du, and the result are each rounded once, sums lose 2^-23 a step
    rel = 3.5 * half(dtype) + (16 + n + 48) * 2.0 ** -23
    for name, y, want in zip(("h", "dx", "dgate", "dup"), got, (a * u, dg @ wg + du @ wu, dg.T @ x, du.T @ x)):
        within(y, want, rel * want.abs(), name)


# ------------------------------------------------------------------------------------------ results in one allocation
def test_writes_to_one_result_are_none_to_another():
    """The two weights' gradients, and the results of clip_gradients, share an allocation."""
    x, wg, wu, dh = glu_inputs(40, 64, 75, BF16, 81)
    gate, up = (t.detach().requires_grad_(True) for t in (wg, wu))
    student.gated_linear_unit(x, gate, up).backward(dh)
    clipped, _ = student.clip_gradients([gate.grad, up.grad], 1e9)
    for a, b in ((gate.grad, up.grad), clipped):
        kept = b.clone()
        p = torch.ones_like(b).requires_grad_(True)
        y = (p * b).sum()  # saves b
        a.add_(1)
        y.backward()
        assert torch.equal(p.grad, kept) and torch.equal(b, kept) and b._version == 0


# ------------------------------------------------------------------------------------------ angles of fp32 tensors
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,head", [(2, 3), (16, 16), (128, 128)])
def test_rotary_fp32_keeps_small_sines(dim, head, layout):
    """Positions whose angles lie close to multiples of pi / 2 (355, 710, 103993, ... for one radian a position):
    cosines and sines near zero are as exact, relatively, as others."""
    cfg = student.RotaryConfig(head, rotary_dim=dim, layout=layout)
    pos = torch.tensor([0, 1, 11, 22, 44, 355, 710, 1065, -355, 103993, 104348, 833719, 1000003], device="cuda")
    q = randn(13, 4, head, seed=1)
    got = student.rotary_embedding(q, q[:, :1], pos, cfg)[0].double()
    angle = pos.double()[:, None, None] * torch.tensor(cfg.frequencies(), dtype=torch.float64, device="cuda")
    ia, ib = ((slice(0, dim // 2), slice(dim // 2, dim)) if layout == "half" else (slice(0, dim, 2), slice(1, dim, 2)))
    a, b, cos, sin = q.double()[..., ia], q.double()[..., ib], angle.cos(), angle.sin()
    # cosine and sine: one unit in the last place, and half of one for the correction; one product is rounded. The
    # frequencies' own rounding and the correction's second order: |p| 2^-52 and 1e-14
    rel, off = 1.5 * 2.0 ** -23 + 2.0 ** -24, pos.double().abs()[:, None, None] * 2.0 ** -52 + 1e-14
    for at, u, v in ((ia, a * cos, -b * sin), (ib, b * cos, a * sin)):
        tol = half(FP32) * (u + v).abs() + rel * (u.abs() + v.abs()) + off * (a.abs() + b.abs())
        assert bool(((got[..., at] - (u + v)).abs() <= tol).all())


def test_ramp_in_the_pair_index_eager_and_compiled():
    cfg = student.RotaryConfig(64, scaling="yarn", factor=8.0, ramp="index")
    q, k = randn(9, 4, 64, seed=1, dtype=BF16), randn(9, 2, 64, seed=2, dtype=BF16)
    pos = torch.arange(9, device="cuda") * 1000
    check_rotary(q, k, pos, cfg)
    fn = lambda q, k: student.rotary_embedding(q, k, pos, cfg)  # noqa: E731
    dy = [randn(*t.shape, seed=3, dtype=BF16) for t in (q, k)]
    results = []
    for f in (fn, torch.compile(fn, fullgraph=True)):
        leaves = [t.detach().requires_grad_(True) for t in (q, k)]
        out = f(*leaves)
        results.append([*out, *torch.autograd.grad(out, leaves, dy)])
    for a, b in zip(*results):
        assert torch.equal(a, b)
    other = student.rotary_embedding(q, k, pos, student.RotaryConfig(64, scaling="yarn", factor=8.0))
    assert not torch.equal(results[0][0], other[0])


# ------------------------------------------------------------------------------------------ no term of a sum is lost
# every forward kernel, whole and partial tiles; one product and K-split ones, whose ranges end inside and at tiles;
# sizes that are no multiple of a tile, a k block, a 16-byte row
@pytest.mark.parametrize("n,h,f", [
    (1, 1000, 2730), (8, 4096, 512), (9, 72, 64), (24, 4096, 1408), (37, 1024, 2816), (64, 4096, 11264), (128, 520, 333),
    (129, 8, 8), (300, 4096, 264), (513, 136, 1025), (1111, 1000, 2730), (1724, 306, 811), (2048, 1024, 2816),
    (4096, 256, 512), (8192, 1024, 2816)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_glu_sums_are_exact_on_integers(n, h, f, dtype):
    check_exact(integers(n, h, seed=1, dtype=dtype, density=0.5), integers(f, h, seed=2, dtype=dtype, density=0.25),
                integers(f, h, seed=3, dtype=dtype, density=0.25), integers(n, f, seed=4, dtype=dtype, density=0.5))


@pytest.mark.parametrize("n,h,f", [(1, 70, 90), (130, 33, 65), (700, 257, 300)])
def test_glu_fp32_sums_are_exact_on_integers(n, h, f):
    check_exact(integers(n, h, seed=1, dtype=FP32, density=0.5), integers(f, h, seed=2, dtype=FP32, density=0.5),
                integers(f, h, seed=3, dtype=FP32, density=0.5), integers(n, f, seed=4, dtype=FP32, density=0.5))


# gates at which e^g (GELU: e^{-g^2 / 2}) stays above the smallest normal number of bf16 and fp32
TAILS = {"silu": 80.0, "gelu": 12.8, "gelu_tanh": 10.0}


@pytest.mark.parametrize("act", list(TAILS))
@pytest.mark.parametrize("n", [5, 40, 300])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_glu_activation_and_derivative_in_their_tails(dtype, n, act):
    """act(g) and act'(g) alone: one element of x is 1, the up product 1. Relative to their values, however small."""
    end = TAILS[act]
    g = torch.cat([torch.linspace(-end, -3, 300, device="cuda"), torch.linspace(3, end, 100, device="cuda")]).to(dtype)
    x = torch.zeros(n, 8, device="cuda", dtype=dtype)
    x[0, 0] = 1
    wg, wu = torch.zeros(2, 400, 8, device="cuda", dtype=dtype)
    wg[:, 0], wu[:, 0] = g, 1
    dh = torch.zeros(n, 400, device="cuda", dtype=dtype)
    dh[0] = 1
    h, _, dgate, dup = glu_pass(x, wg, wu, act, dh)
    v = g.double()
    if act == "silu":
        s = 1 / (1 + torch.exp(-v))
        a, d = v * s, s * (1 + v * (1 - s))
    elif act == "gelu":
        cdf = torch.special.erfc(-v / math.sqrt(2)) / 2
        a, d = v * cdf, cdf + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    else:
        z = 2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)
        s, t = 1 / (1 + torch.exp(-z)), 1 / (1 + torch.exp(z))
        a, d = v * s, s + v * s * t * 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * v * v)
    # e^x of |x| <= 88 in fp32: x and x log2(e) are each rounded (2^-18 of 88 or 127), z of three more roundings;
    # in d the two terms may cancel down to a tenth of the larger
    rel = half(dtype) + 2.0 ** -15
    within(h[0], a, rel * a.abs(), "act")
    within(dgate[:, 0], d, (half(dtype) + 2.0 ** -14) * d.abs(), "derivative")
    within(dup[:, 0], a, rel * a.abs(), "act in the backward pass")


@pytest.mark.parametrize("value,max_norm", [(1e37, 1e-2), (3e38, 0.1), (1e38, 1e-6), (1e38, 0.0)])
def test_clip_by_factors_below_the_normal_range(value, max_norm):
    """A diverged step's gradients: the factor is no normal fp32 number, the clipped values are."""
    for dtype in (FP32, BF16):
        g = torch.full((1000,), value, device="cuda", dtype=dtype)
        g[::3] *= -0.5
        want = g.double() * (max_norm / (float(g.double().square().sum().sqrt()) + 1e-6))
        clipped, _ = student.clip_gradients([g], max_norm)
        # the factor, two products (the second by a power of two), the value
        within(clipped[0], want, (half(dtype) + 2 * half(FP32)) * want.abs())
        student.clip_grad_norm_(_params(g), max_norm)
        assert torch.equal(g, clipped[0])


# ------------------------------------------------------------------------------------------ the custom ops as such
def _custom_op_calls():
    ops = torch.ops.orda_b200
    for n, h, f in ((40, 64, 72), (3, 66, 75), (0, 64, 72), (300, 64, 71)):
        x, wg, wu, _ = glu_inputs(n, h, f, BF16, 5)
        yield ops.glu_forward, (*(t.requires_grad_(True) for t in (x, wg, wu)), 0)
    cfg = student._config_values(student.RotaryConfig(64, rotary_dim=32))
    q, k, pos = randn(2, 5, 4, 64, seed=1), randn(2, 2, 5, 64, seed=2).transpose(1, 2), torch.arange(5, device="cuda")
    w = [randn(64, seed=3 + i).requires_grad_(True) for i in range(2)]
    q, k = q.requires_grad_(True), k.requires_grad_(True)
    yield ops.rotary, (q, k, pos, None, None, 0.0, False, *cfg)
    yield ops.rotary, (q, k, pos, *w, 1e-6, False, *cfg)


@pytest.mark.parametrize("which", range(6))
def test_custom_ops_keep_the_rules_of_custom_ops(which):
    """Schema, shapes without data, autograd registration, and tracing with dynamic shapes."""
    op, args = list(_custom_op_calls())[which]
    torch.library.opcheck(op, args)


@pytest.mark.parametrize("which", ["glu", "rotary", "norm"])
def test_captured_backward_of_a_recorded_call_is_refused_as_a_plain_one_is(which):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Pass(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    x, wg, wu, q, k, wq, wk, pos = _block_inputs(4)
    cfg = student.RotaryConfig(64)
    call = {"glu": lambda t: student.gated_linear_unit(x, t, wu),
            "rotary": lambda t: student.rotary_embedding(t, k, pos, cfg)[0],
            "norm": lambda t: student.qk_norm_rotary(t, k, wq, wk, pos, cfg)[0]}[which]
    leaf = (wg if which == "glu" else q).detach().requires_grad_(True)

    def step():
        with Pass():
            y = call(leaf)
            return torch.autograd.grad(y, leaf, torch.ones_like(y))[0]

    want = step().clone()
    eager = call(leaf)  # recorded on the default stream
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="still lives"):
        with torch.cuda.graph(graph):
            step()
    del eager, graph
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    assert torch.equal(got, want)


# ------------------------------------------------------------------------------------------ results behind 2^31 elements
@pytest.mark.parametrize("norm", [False, True])
def test_rotary_results_and_gradients_behind_32_bits(norm):
    """Tokens whose results, and whose gradients, lie behind 2^31 elements, against the same tokens alone."""
    n, heads, d = 70_000, 256, 128
    assert n * heads * d > 2 ** 31
    cfg, pos = student.RotaryConfig(d), torch.arange(n, device="cuda")
    w = [(1 + randn(d, seed=i, scale=0.1)).requires_grad_(norm) for i in range(2)]
    rows = torch.tensor([0, 65_535, 65_536, n - 1], device="cuda")  # 65536 x 256 x 128 = 2^31
    values, dys = randn(4, heads, d, seed=3, dtype=BF16), randn(4, heads, d, seed=4, dtype=BF16)

    def run(q, k, p, dy):
        q = q.requires_grad_(True)
        out = (student.qk_norm_rotary(q, k, *w, p, cfg) if norm else student.rotary_embedding(q, k, p, cfg))[0]
        return out.detach(), *torch.autograd.grad(out, [q, *w[:1]] if norm else [q], dy)

    q = torch.ones(n, heads, d, device="cuda", dtype=BF16)
    dy = torch.zeros_like(q)
    q[rows], dy[rows] = values, dys
    got = run(q, torch.ones(n, 1, d, device="cuda", dtype=BF16), pos, dy)
    want = run(values, torch.ones(4, 1, d, device="cuda", dtype=BF16), pos[rows], dys)
    assert torch.equal(got[0][rows], want[0]) and torch.equal(got[1][rows], want[1])
    got[1][rows] = 0
    assert not got[1].any()
    if norm:  # the other tokens add zeros, in another order of the same terms
        torch.testing.assert_close(got[2], want[2], rtol=0, atol=float(want[2].abs().max()) * 4 * heads * 2.0 ** -24)
