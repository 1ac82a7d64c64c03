"""GPU tests of ``orda_ce_kernel.student`` against plain 64-bit formulas.

Tolerances are worked out per element before anything runs: ``half`` is the largest relative error of one
rounding to the tensors' type (half a unit in the last place), a sum of n products formed in fp32 is off
by at most ``n 2^-23`` of the sum of their magnitudes (tensor-core accumulators may truncate, 2^-23 a
step), and what an intermediate rounding to 16 bits moves is carried through the formula that reads it.
"""
from __future__ import annotations

import math

import pytest
import torch

from orda_ce_kernel import _native, student

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def half(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def randn(*shape, seed, dtype=FP32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def within(got, want, tol, what=""):
    """|got - want| <= tol everywhere; a value that the type cannot hold may be off by its smallest step."""
    assert got.shape == want.shape, (what, got.shape, want.shape)
    got, want = got.detach(), want.detach()
    off = (got.double() - want).abs() - (tol + torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps)
    assert not torch.isnan(got).any(), what
    worst = float(off.max()) if off.numel() else 0.0
    assert worst <= 0, (what, worst, float((got.double() - want).abs().max()))


# ------------------------------------------------------------------------------------------ gated feed-forward block
def act64(name, g):
    """act, act' in 64 bits."""
    g = g.detach().requires_grad_(True)
    if name == "silu":
        a = g * torch.sigmoid(g)
    elif name == "relu":
        a = torch.relu(g)
    elif name == "gelu":
        a = torch.nn.functional.gelu(g)
    else:
        a = torch.nn.functional.gelu(g, approximate="tanh")
    return a.detach(), torch.autograd.grad(a.sum(), g)[0]


def glu64(x, wg, wu, act, dh=None):
    """{name: (value, tolerance)} of h and, with dh, the gradients."""
    dt, k = x.dtype, x.shape[1]
    hf = half(dt)
    sub = torch.finfo(dt).smallest_normal * hf  # the same below the normal range: half of the smallest step
    x, wg, wu = x.double(), wg.double(), wu.double()
    g, u = x @ wg.T, x @ wu.T
    eg, eu = (x.abs() @ w.abs().T * (k * 2.0 ** -23) for w in (wg, wu))  # of the products
    a, d = act64(act, g)
    h = a * u
    # |act'| <= 1.13; the activation itself is off by at most 2^-18 of |g| (its exponential 2^-21, its quotient 2^-21)
    ea = 1.13 * eg + 2.0 ** -18 * g.abs()
    out = {"h": (h, hf * h.abs() + (ea * (u.abs() + eu) + a.abs() * eu) * (1 + hf))}
    if dh is None:
        return out
    dh = dh.double()
    # what the backward pass reads: g and u rounded (16-bit types)
    rg, ru = eg + hf * g.abs() + sub, eu + hf * u.abs() + sub
    # |act''| <= 1.13 (relu: its slope jumps within eg of 0)
    ed = 1.13 * rg + 2.0 ** -17 * (1 + g.abs()) if act != "relu" else (g.abs() <= eg).double()
    dg, du = dh * u * d, dh * a
    edg = dh.abs() * (ru * (d.abs() + ed) + u.abs() * ed)
    edu = dh.abs() * (1.13 * rg + 2.0 ** -18 * g.abs())
    edg, edu = edg + hf * (dg.abs() + edg) + sub, edu + hf * (du.abs() + edu) + sub  # dg and du are rounded too
    mg, mu = dg.abs() + edg, du.abs() + edu

    def grad(v, err, magnitude, n):
        return v, hf * v.abs() + (err + magnitude * (n * 2.0 ** -23)) * (1 + hf)

    n, f = dh.shape
    out["dx"] = grad(dg @ wg + du @ wu, edg @ wg.abs() + edu @ wu.abs(), mg @ wg.abs() + mu @ wu.abs(), 2 * f + 8)
    out["dgate"] = grad(dg.T @ x, edg.T @ x.abs(), mg.T @ x.abs(), n + 8)
    out["dup"] = grad(du.T @ x, edu.T @ x.abs(), mu.T @ x.abs(), n + 8)
    return out


def glu_inputs(n, h, f, dtype, seed):
    return (randn(n, h, seed=seed, dtype=dtype), randn(f, h, seed=seed + 1, dtype=dtype, scale=h ** -0.5),
            randn(f, h, seed=seed + 2, dtype=dtype, scale=h ** -0.5), randn(n, f, seed=seed + 3, dtype=dtype, scale=0.1))


def check_glu(x, wg, wu, dh, act):
    want = glu64(x, wg, wu, act, dh)
    with torch.no_grad():
        h = student.gated_linear_unit(x, wg, wu, activation=act)
    within(h, *want["h"], "h")
    leaves = [t.detach().requires_grad_(True) for t in (x, wg, wu)]
    h = student.gated_linear_unit(*leaves, activation=act)
    assert h.is_contiguous()
    within(h, *want["h"], "h of the training pass")
    for name, g in zip(("dx", "dgate", "dup"), torch.autograd.grad(h, leaves, dh)):
        within(g, *want[name], name)


# rows: one, the few-rows kernel's blocks of 8, both sides of its limit, partial and whole 512-row tiles
@pytest.mark.parametrize("n", [1, 2, 8, 9, 16, 17, 32, 33, 130, 512, 700])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_glu_rows(n, dtype):
    check_glu(*glu_inputs(n, 192, 200, dtype, n), "silu")


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("n", [5, 300])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_glu_activations(act, n, dtype):
    check_glu(*glu_inputs(n, 136, 264, dtype, 7), act)


# hidden and ffn sizes that end inside tiles, k blocks, 16-byte rows
@pytest.mark.parametrize("h,f", [(1, 1), (7, 9), (8, 16), (24, 1), (65, 127), (64, 128), (129, 130), (1000, 61)])
@pytest.mark.parametrize("n", [3, 65])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_glu_odd_sizes(h, f, n, dtype):
    check_glu(*glu_inputs(n, h, f, dtype, 11), "silu")


@pytest.mark.parametrize("shape", [(2048, 1024, 2816), (1111, 1000, 2730), (24, 4096, 1408), (4096, 256, 512)])
def test_glu_larger(shape):
    """Several waves of tiles, the K-split gradients, a batch of decoded tokens."""
    check_glu(*glu_inputs(*shape, BF16, 3), "silu")


@pytest.mark.parametrize("n", [4, 200])
def test_glu_strided_operands(n):
    """Slices of wider tensors: read in place where rows are aligned, copied where not; the gradients keep
    the operands' shapes."""
    big = randn(n, 400, seed=1, dtype=BF16)
    wide = randn(2, 96, 160, seed=2, dtype=BF16, scale=0.1)
    for x, wg, wu in ((big[:, 8:136], wide[0, :, :128], wide[1, :, 16:144]),   # aligned slices
                      (big[:, 3:131], wide[0, :, 1:129], wide[1, :, :128]),    # not aligned
                      (randn(128, n, seed=4, dtype=BF16).T, wide[0, :, :128], wide[1, :, :128])):  # transposed
        check_glu(x, wg, wu, randn(n, 96, seed=5, dtype=BF16), "gelu")


def test_glu_leading_dimensions_and_partial_gradients():
    x, wg, wu, dh = glu_inputs(60, 64, 72, BF16, 21)
    want = glu64(x, wg, wu, "silu", dh)
    for need in ((True, False, False), (False, True, False), (False, False, True), (True, False, True)):
        leaves = [t.detach().requires_grad_(r) for t, r in zip((x, wg, wu), need)]
        h = student.gated_linear_unit(leaves[0].view(3, 4, 5, 64), leaves[1], leaves[2])
        assert h.shape == (3, 4, 5, 72)
        h.backward(dh.view_as(h))
        for t, r, name in zip(leaves, need, ("dx", "dgate", "dup")):
            assert (t.grad is not None) == r
            if r:
                within(t.grad, *want[name], name)
    one = student.gated_linear_unit(x[0], wg, wu)  # a single vector
    within(one, want["h"][0][0], want["h"][1][0])
    # a broadcast gradient (the sum's) and one that arrives transposed
    leaf = x.detach().requires_grad_(True)
    student.gated_linear_unit(leaf, wg, wu).sum().backward()
    within(leaf.grad, *glu64(x, wg, wu, "silu", torch.ones_like(dh))["dx"])
    leaf.grad = None
    student.gated_linear_unit(leaf, wg, wu).backward(dh.T.contiguous().T)
    within(leaf.grad, *want["dx"])


# each forward kernel: rows at a time, weights first, 256-row and 512-row tiles, fp32
@pytest.mark.parametrize("n,h,f,dtype", [(5, 64, 72, BF16), (40, 64, 72, BF16), (140, 64, 72, BF16), (140, 64, 71, BF16),
                                         (512, 4096, 9470, BF16), (20, 64, 72, FP32)])
def test_c_glu_results_that_start_at_any_element(n, h, f, dtype):
    """h (and its gradient dh) one element behind a boundary, with even and odd row strides, between values
    that have to stay."""
    x, wg, wu, dh = glu_inputs(n, h, f, dtype, 31)
    leaves = [t.detach().requires_grad_(True) for t in (x, wg, wu)]
    want = student.gated_linear_unit(*leaves)
    want_dx, want_dg, want_du = torch.autograd.grad(want, leaves, dh)
    lib, fp = _native.load(), (f + 7) // 8 * 8
    code = {BF16: _native.BF16, FP32: _native.F32}[dtype]
    stream = torch.cuda.current_stream().cuda_stream
    for ld in (f + f % 2, f + 1 - f % 2):  # even, odd
        for start in (1, 2):
            buf, gbuf = (torch.full((start + n * ld + 1,), 7.0, device="cuda", dtype=dtype) for _ in range(2))
            rows = buf[start:start + n * ld].view(n, ld)
            gbuf[start:start + n * ld].view(n, ld)[:, :f] = dh
            pre = torch.empty(2, n, fp, device="cuda", dtype=dtype)
            status = torch.zeros(1, device="cuda", dtype=torch.int32)
            dx, dw = torch.empty(n, h, device="cuda", dtype=dtype), torch.empty(fp + f, h, device="cuda", dtype=dtype)
            size = buf.element_size()
            a = _native.GluArgs(abi_version=_native.ABI_VERSION, dtype=code, activation=_native.ACT_SILU, rows=n, hidden=h,
                                ffn=f, x=x.data_ptr(), ld_x=h, gate=wg.data_ptr(), ld_gate=h, up=wu.data_ptr(), ld_up=h,
                                h=buf.data_ptr() + start * size, ld_h=ld, pre_gate=pre[0].data_ptr(), ld_pre=fp,
                                pre_up=pre[1].data_ptr(), grad_cols=h, dh=gbuf.data_ptr() + start * size,
                                dx=dx.data_ptr(), dweights=dw.data_ptr(), device_status=status.data_ptr())
            assert lib.orda_glu_forward(a, stream) == _native.OK
            assert torch.equal(rows[:, :f], want) and bool((rows[:, f:] == 7).all())
            assert bool((buf[:start] == 7).all()) and float(buf[-1]) == 7.0
            need = lib.orda_glu_backward_workspace_bytes(a)
            ws = torch.empty(need, device="cuda", dtype=torch.uint8)
            assert lib.orda_glu_backward(a, ws.data_ptr(), need, stream) == _native.OK
            assert torch.equal(dx, want_dx) and torch.equal(dw[:f], want_dg) and torch.equal(dw[fp:], want_du)
            assert not status.any()


def test_glu_no_rows():
    wg = randn(24, 16, seed=1, dtype=BF16).requires_grad_(True)
    x = torch.empty(0, 16, device="cuda", dtype=BF16, requires_grad=True)
    h = student.gated_linear_unit(x, wg, wg.detach())
    assert h.shape == (0, 24)
    h.sum().backward()
    assert x.grad.shape == x.shape and not wg.grad.any()


def test_glu_same_weight_twice_and_autocast():
    x, wg, _, dh = glu_inputs(40, 64, 72, BF16, 31)
    w = wg.detach().requires_grad_(True)
    student.gated_linear_unit(x, w, w).backward(dh)
    want = glu64(x, wg, wg, "silu", dh)
    total = want["dgate"][0] + want["dup"][0]
    # two rounded gradients, added and rounded once more
    within(w.grad, total, (want["dgate"][1] + want["dup"][1]) * (1 + half(BF16)) + half(BF16) * total.abs())
    x32, w32 = x.float().requires_grad_(True), wg.float().requires_grad_(True)
    with torch.autocast("cuda", dtype=BF16):
        h = student.gated_linear_unit(x32, w32, w32)
    assert h.dtype == BF16
    within(h, *want["h"])
    h.backward(dh)
    assert x32.grad.dtype == FP32 and w32.grad.dtype == FP32
    within(x32.grad.to(BF16), *want["dx"])


def test_glu_values_that_are_not_finite_stay_in_their_rows():
    x, wg, wu, _ = glu_inputs(600, 64, 72, BF16, 41)
    clean = student.gated_linear_unit(x, wg, wu)
    for rows in (slice(0, 5), slice(0, 600)):  # few-rows kernel, pair GEMM
        y = x[rows].clone()
        y[3] = float("nan")
        h = student.gated_linear_unit(y, wg, wu)
        assert torch.isnan(h[3]).all()
        keep = torch.arange(y.shape[0], device="cuda") != 3
        ref = clean[rows][keep] if y.shape[0] > 32 else student.gated_linear_unit(x[rows], wg, wu)[keep]
        assert torch.equal(h[keep], ref)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_glu_gradient_against_differences(act):
    x, wg, wu, dh = glu_inputs(6, 24, 16, FP32, 51)
    leaves = [t.requires_grad_(True) for t in (x, wg, wu)]
    grads = torch.autograd.grad(student.gated_linear_unit(*leaves, activation=act), leaves, dh)
    for i, g in enumerate(grads):
        v = randn(*g.shape, seed=60 + i)
        step = 2.0 ** -7  # error step^2 of the quotient, fp32 noise 2^-24 / step
        with torch.no_grad():
            up, down = ([t + s * step * v if j == i else t for j, t in enumerate(leaves)] for s in (1, -1))
            diff = ((student.gated_linear_unit(*up, activation=act) - student.gated_linear_unit(*down, activation=act))
                    .double() * dh.double()).sum() / (2 * step)
        scale = float((g.double().abs() * v.double().abs()).sum())
        assert abs(float((g.double() * v.double()).sum()) - float(diff)) <= scale * (step ** 2 * 4 + 2.0 ** -14)


# ------------------------------------------------------------------------------------------ rotary positions
def turn64(x, positions, cfg, inverse=False):
    """(rotated values, magnitudes of the two terms of each) in 64 bits. x [..., heads, D]."""
    x = x.double()
    angle = positions.double()[..., None] * torch.tensor(cfg.frequencies(), dtype=torch.float64, device=x.device)
    cos, sin = torch.cos(angle)[..., None, :] * cfg.value_scale, torch.sin(angle)[..., None, :] * cfg.value_scale
    if inverse:
        sin = -sin
    r = cfg.dim
    y, size = x.clone(), x.abs()
    ia, ib = ((slice(0, r // 2), slice(r // 2, r)) if cfg.layout == "half" else (slice(0, r, 2), slice(1, r, 2)))
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * cos - b * sin, b * cos + a * sin
    size = size.clone()
    size[..., ia] = size[..., ib] = (a.abs() + b.abs()) * cfg.value_scale
    return y, size


# a turn's angle is off by less than 2e-7 in 32-bit turns, cosine and sine by 2^-22, three roundings of 2^-24
TURN = 1e-6


def check_rotary(q, k, pos, cfg):
    dt = q.dtype
    leaves = [q.detach().requires_grad_(True), k.detach().requires_grad_(True)]
    full = pos if pos.ndim == q.ndim - 2 else pos.expand(q.shape[:-2])
    out = student.rotary_embedding(*leaves, pos, cfg)
    dy = [randn(*t.shape, seed=70 + i, dtype=dt) for i, t in enumerate(out)]
    grads = torch.autograd.grad(out, leaves, dy)
    for x, y, d, g in zip((q, k), out, dy, grads):
        assert y.is_contiguous()
        want, size = turn64(x, full, cfg)
        within(y, want, half(dt) * want.abs() + TURN * size, "y")
        want, size = turn64(d, full, cfg, inverse=True)
        within(g, want, half(dt) * want.abs() + TURN * size, "gradient")


CONFIGS = [
    dict(head_dim=128), dict(head_dim=128, layout="interleaved"),
    dict(head_dim=64, rotary_dim=32), dict(head_dim=64, rotary_dim=32, layout="interleaved"),
    dict(head_dim=80), dict(head_dim=80, rotary_dim=20, layout="interleaved"), dict(head_dim=80, rotary_dim=48),
    dict(head_dim=512), dict(head_dim=512, rotary_dim=6, layout="interleaved"), dict(head_dim=256, rotary_dim=64),
    dict(head_dim=2), dict(head_dim=3, rotary_dim=2), dict(head_dim=37, rotary_dim=22, layout="interleaved"),
    dict(head_dim=50), dict(head_dim=100, rotary_dim=100, layout="interleaved"), dict(head_dim=511, rotary_dim=510),
]


@pytest.mark.parametrize("cfg", CONFIGS, ids=lambda c: "-".join(str(v) for v in c.values()))
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_rotary_head_shapes(cfg, dtype):
    d = cfg["head_dim"]
    q, k = randn(2, 9, 6, d, seed=1, dtype=dtype), randn(2, 9, 3, d, seed=2, dtype=dtype)
    check_rotary(q, k, torch.arange(9, device="cuda"), student.RotaryConfig(**cfg))


@pytest.mark.parametrize("scaling", ["none", "linear", "ntk", "yarn"])
@pytest.mark.parametrize("ints", [torch.int32, torch.int64])
def test_rotary_far_and_negative_positions(scaling, ints):
    cfg = student.RotaryConfig(64, scaling=scaling, factor=1.0 if scaling == "none" else 8.0)
    pos = torch.tensor([0, 1, -1, 1000003, 2 ** 31 - 1, -(2 ** 31), 7, 7], device="cuda", dtype=ints)
    check_rotary(randn(8, 4, 64, seed=3, dtype=FP32), randn(8, 1, 64, seed=4, dtype=FP32), pos, cfg)


@pytest.mark.parametrize("heads", [(1, 1), (33, 1), (5, 7), (40, 8)])
@pytest.mark.parametrize("tokens", [1, 3, 700])
def test_rotary_heads_and_tokens(heads, tokens):
    q, k = (randn(tokens, h, 128, seed=h, dtype=BF16) for h in heads)
    pos = torch.randint(0, 9000, (tokens,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    check_rotary(q, k, pos, student.RotaryConfig(128))


def test_rotary_strides():
    b, t, hq, hk, d = 2, 7, 4, 2, 64
    cfg = student.RotaryConfig(d, rotary_dim=32)
    qkv = randn(b, t, (hq + 2 * hk) * d + 3, seed=5, dtype=BF16)
    pos = torch.randint(0, 500, (t, b), device="cuda").T  # strided positions
    views = [(qkv[..., o: o + hq * d].unflatten(-1, (hq, d)), qkv[..., o + hq * d: o + (hq + hk) * d].unflatten(-1, (hk, d)))
             for o in (0, 1, 3)]  # aligned and unaligned slices of a fused projection (odd row length)
    even = randn(b, t, (hq + 2 * hk) * d, seed=5, dtype=BF16)
    views.append((even[..., : hq * d].view(b, t, hq, d), even[..., hq * d: (hq + hk) * d].view(b, t, hk, d)))
    views.append((randn(b, hq, t, d, seed=6, dtype=BF16).transpose(1, 2), randn(b, hk, t, d, seed=7, dtype=BF16).transpose(1, 2)))
    views.append((randn(b, t, d, hq, seed=8, dtype=BF16).transpose(2, 3), randn(b, t, 1, d, seed=9, dtype=BF16).expand(b, t, hk, d)))
    for q, k in views:
        check_rotary(q, k, pos, cfg)
    # gradients that arrive strided and broadcast
    q = views[3][0].detach().requires_grad_(True)
    k = views[3][1].detach().requires_grad_(True)
    oq, ok_ = student.rotary_embedding(q, k, pos, cfg)
    dy = randn(b, hq, t, d, seed=10, dtype=BF16).transpose(1, 2)
    gq, gk = torch.autograd.grad([oq, ok_.sum()], [q, k], [dy, torch.ones((), device="cuda", dtype=BF16)])
    for g, d_ in ((gq, dy), (gk, torch.ones(b, t, hk, d, device="cuda", dtype=BF16))):
        want, size = turn64(d_, pos, cfg, inverse=True)
        within(g, want, half(BF16) * want.abs() + TURN * size)
    # only one of the two results is used
    (only,) = torch.autograd.grad(student.rotary_embedding(q, k, pos, cfg)[0], [q], dy)
    assert torch.equal(only, gq)


PARTIAL = [dict(head_dim=64, rotary_dim=32), dict(head_dim=80, rotary_dim=20, layout="interleaved"),
           dict(head_dim=3, rotary_dim=2), dict(head_dim=37, rotary_dim=22, layout="interleaved"),
           dict(head_dim=512, rotary_dim=6), dict(head_dim=256, rotary_dim=64)]


@pytest.mark.parametrize("cfg", PARTIAL, ids=lambda c: "-".join(str(v) for v in c.values()))
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_values_that_are_not_finite_pass_through_alone(cfg, dtype):
    d, r = cfg["head_dim"], cfg["rotary_dim"]
    cfg, pos = student.RotaryConfig(**cfg), torch.arange(1, 6, device="cuda")
    clean = randn(5, 3, d, seed=14, dtype=dtype)
    x = clean.clone()
    x[0, 0, r], x[1, 1, d - 1], x[2, 2, (r + d) // 2] = math.inf, -math.inf, math.nan
    leaf = clean.clone().requires_grad_(True)
    y, want = student.rotary_embedding(x, x, pos, cfg)[0], student.rotary_embedding(leaf, clean, pos, cfg)[0]
    assert torch.equal(y[..., :r], want[..., :r])
    torch.testing.assert_close(y[..., r:], x[..., r:], rtol=0, atol=0, equal_nan=True)
    (g,) = torch.autograd.grad(want, leaf, x)
    torch.testing.assert_close(g[..., r:], x[..., r:], rtol=0, atol=0, equal_nan=True)
    assert bool(torch.isfinite(g[..., :r]).all())
    # with the norm: a head whose mean square is infinite is zero but for that element
    w = (1 + randn(d, seed=15, scale=0.1)).requires_grad_(True)
    bad = clean.clone()
    bad[0, 0, r] = math.inf
    y = student.qk_norm_rotary(bad, clean, w, w, pos, cfg)[0].detach()
    want = student.qk_norm_rotary(clean, clean, w, w, pos, cfg)[0]
    lost = torch.zeros(5, 3, d, device="cuda", dtype=torch.bool)
    lost[0, 0, r] = True
    assert bool(torch.isnan(y[lost]).all()) and not y[0, 0][~lost[0, 0]].any()
    y[0, 0] = want[0, 0].detach()
    assert torch.equal(y, want)
    # a gradient that is not finite reaches one element of the weight's
    dy = clean.clone()
    dy[1, 1, d - 1] = math.inf
    (gw,) = torch.autograd.grad(want, w, dy)
    assert not bool(torch.isfinite(gw[d - 1])) and bool(torch.isfinite(gw[:d - 1]).all())


def test_rotary_no_tokens_and_no_heads():
    cfg = student.RotaryConfig(64)
    q, k = student.rotary_embedding(randn(0, 4, 64, seed=1), randn(0, 2, 64, seed=1),
                                    torch.zeros(0, device="cuda", dtype=torch.long), cfg)
    assert q.shape == (0, 4, 64) and k.shape == (0, 2, 64)
    q = randn(3, 4, 64, seed=1)
    pos = torch.arange(3, device="cuda")
    got, none = student.rotary_embedding(q, q[:, :0], pos, cfg)
    assert none.shape == (3, 0, 64)
    assert torch.equal(got, student.rotary_embedding(q, q, pos, cfg)[0])


# ------------------------------------------------------------------------------------------ norms with the rotation
def check_qk_norm(q, k, wq, wk, pos, cfg, eps=1e-6):
    dt, d = q.dtype, q.shape[-1]
    full = pos if pos.ndim == q.ndim - 2 else pos.expand(q.shape[:-2])
    leaves = [t.detach().requires_grad_(True) for t in (q, k, wq, wk)]
    out = student.qk_norm_rotary(*leaves, pos, cfg, eps)
    dy = [randn(*t.shape, seed=80 + i, dtype=dt) for i, t in enumerate(out)]
    grads = torch.autograd.grad(out, leaves, dy)
    with torch.no_grad():
        for a, b in zip(student.qk_norm_rotary(q, k, wq, wk, pos, cfg, eps), out):
            assert torch.equal(a, b)
    rel = d * 2.0 ** -24 + 2.0 ** -21  # of the norm: d positive terms added in fp32, one rsqrt, a few roundings
    for x, w, y, e, gx, gw in zip((q, k), (wq, wk), out, dy, grads[:2], grads[2:]):
        x, w64 = x.double(), w.double()
        r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
        n = x * r
        want, size = turn64(n * w64, full, cfg)
        within(y, want, half(dt) * want.abs() + (TURN + rel) * size, "y")
        z, zsize = turn64(e, full, cfg, inverse=True)
        count = x.numel() // d
        want = (z * n).flatten(0, -2).sum(0)
        within(gw, want, half(w.dtype) * want.abs()
               + (TURN + rel + (count + 8) * 2.0 ** -24) * (zsize * n.abs()).flatten(0, -2).sum(0), "dweight")
        t, tsize = z * w64, zsize * w64.abs()
        want = r * (t - n * (t * n).mean(-1, keepdim=True))
        within(gx, want, half(dt) * want.abs()
               + (2 * TURN + 4 * rel) * r * (tsize + n.abs() * (tsize * n.abs()).mean(-1, keepdim=True)), "dx")


@pytest.mark.parametrize("cfg", CONFIGS, ids=lambda c: "-".join(str(v) for v in c.values()))
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_qk_norm_head_shapes(cfg, dtype):
    d = cfg["head_dim"]
    q, k = randn(2, 9, 6, d, seed=1, dtype=dtype), randn(2, 9, 3, d, seed=2, dtype=dtype)
    w = [(1 + randn(d, seed=3 + i, scale=0.2)).to(dtype) for i in range(2)]
    check_qk_norm(q, k, *w, torch.arange(9, device="cuda"), student.RotaryConfig(**cfg))


@pytest.mark.parametrize("heads", [(1, 1), (33, 1), (5, 7), (32, 8)])
@pytest.mark.parametrize("tokens", [1, 3, 1500])
def test_qk_norm_heads_and_tokens(heads, tokens):
    q, k = (randn(tokens, h, 128, seed=h, dtype=BF16) for h in heads)
    w = [1 + randn(128, seed=3 + i, scale=0.2) for i in range(2)]  # fp32 weights of bf16 heads
    check_qk_norm(q, k, *w, torch.arange(tokens, device="cuda", dtype=torch.int32), student.RotaryConfig(128))


def test_qk_norm_strides_and_small_heads():
    b, t, hq, hk, d = 2, 5, 4, 2, 64
    qkv = randn(b, t, (hq + 2 * hk) * d, seed=5, dtype=BF16)
    q, k = qkv[..., : hq * d].view(b, t, hq, d), qkv[..., hq * d: (hq + hk) * d].view(b, t, hk, d)
    w = randn(2, 2 * d, seed=6, dtype=BF16)
    cfg = student.RotaryConfig(d, layout="interleaved", scaling="yarn", factor=4.0)
    check_qk_norm(q, k, w[0, ::2], w[1, 1::2], torch.arange(t, device="cuda"), cfg, eps=1e-2)
    # heads of zeros: the norm is eps alone
    q = q.clone()
    q[:, 1] = 0
    check_qk_norm(q, k, w[0, :d], w[1, :d], torch.arange(t, device="cuda"), cfg, eps=1e-2)
    # the same where the cube of their factor, 1e15, is no fp32 number
    check_qk_norm(q.float(), k.float(), w[0, :d], w[1, :d], torch.arange(t, device="cuda"), cfg, eps=1e-30)


def test_qk_norm_no_tokens():
    cfg = student.RotaryConfig(64)
    w = torch.ones(64, device="cuda", requires_grad=True)
    q, k = student.qk_norm_rotary(randn(0, 4, 64, seed=1), randn(0, 2, 64, seed=1), w, w,
                                  torch.zeros(0, device="cuda", dtype=torch.long), cfg)
    (q.sum() + k.sum()).backward()
    assert not w.grad.any()


def test_qk_norm_gradient_against_differences():
    cfg = student.RotaryConfig(16, rotary_dim=8)
    pos = torch.tensor([3, 9, 100], device="cuda")
    leaves = [randn(3, 2, 16, seed=1), randn(3, 1, 16, seed=2), 1 + randn(16, seed=3, scale=0.1), 1 + randn(16, seed=4, scale=0.1)]
    leaves = [t.requires_grad_(True) for t in leaves]
    dy = [randn(3, 2, 16, seed=5), randn(3, 1, 16, seed=6)]
    grads = torch.autograd.grad(student.qk_norm_rotary(*leaves, pos, cfg), leaves, dy)

    def value(args):
        with torch.no_grad():
            return sum(float((y.double() * d.double()).sum()) for y, d in zip(student.qk_norm_rotary(*args, pos, cfg), dy))

    for i, g in enumerate(grads):
        v = randn(*g.shape, seed=90 + i)
        step = 2.0 ** -8
        diff = (value([t + step * v if j == i else t for j, t in enumerate(leaves)])
                - value([t - step * v if j == i else t for j, t in enumerate(leaves)])) / (2 * step)
        scale = float((g.double().abs() * v.double().abs()).sum()) + float(v.double().abs().sum())
        assert abs(float((g.double() * v.double()).sum()) - diff) <= scale * (step ** 2 * 16 + 2.0 ** -14)


# ------------------------------------------------------------------------------------------ norm and clipping
def clip64(grads, max_norm, eps=1e-6):
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    return norm, min(1.0, max_norm / (norm + eps))


def check_clip(grads, max_norm):
    norm, factor = clip64(grads, max_norm)
    before = [g.clone() for g in grads]
    assert float(student.grad_norm(grads)) == pytest.approx(norm, rel=2.0 ** -23)
    clipped, got = student.clip_gradients(grads, max_norm)
    assert got.shape == () and got.dtype == FP32 and float(got) == pytest.approx(norm, rel=2.0 ** -23)
    params = []
    for g, b in zip(grads, before):
        assert torch.equal(g, b)  # clip_gradients leaves them
        p = torch.nn.Parameter(torch.empty_like(g))
        p.grad = g
        params.append(p)
    for c, b in zip(clipped, before):
        want = b.double() * factor
        assert c.dtype == b.dtype
        # the factor and the product are rounded to fp32, the value to its type
        within(c, want, want.abs() * (half(b.dtype) + 2.0 ** -22))
    params.append(torch.nn.Parameter(torch.ones(3, device="cuda")))  # without a gradient
    assert torch.equal(student.clip_grad_norm_(params, max_norm), got)
    for p, c in zip(params, clipped):
        assert torch.equal(p.grad, c)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("max_norm", [0.0, 0.5, 1e6])
def test_clip_sizes(dtype, max_norm):
    sizes = [(1,), (7,), (8,), (2047,), (2048,), (2049,), (0,), (33, 65), (300, 1001), ()]
    check_clip([randn(*s, seed=i, dtype=dtype) for i, s in enumerate(sizes)], max_norm)


def test_clip_mixed_types_strides_and_alignment():
    flat = randn(5000, seed=1, dtype=BF16)
    grads = [flat[1:1000], flat[1008:2000], randn(64, 33, seed=2).T, randn(40, 50, seed=3, dtype=FP16)[:, ::2],
             randn(3, 5, 7, seed=4).permute(2, 0, 1), randn(100, seed=5)[::3], randn(1, 9, seed=6)]
    check_clip(grads, 1.0)


@pytest.mark.parametrize("count", [95, 96, 97, 768, 769, 1700])
def test_clip_many_tensors(count):
    check_clip([randn(1 + 37 * i % 300, seed=i, dtype=(FP32, BF16, FP16)[i % 3]) for i in range(count)], 1.0)


def test_clip_large():
    check_clip([randn(40_000_000, seed=1, dtype=BF16), randn(3, seed=2), randn(9_999_999, seed=3)], 1.0)


def test_clip_extreme_values():
    for value in (1e30, 1e-30):  # squares behind fp32's range at both ends
        g = torch.full((1000,), value, device="cuda")
        assert float(student.grad_norm([g])) == pytest.approx(value * math.sqrt(1000), rel=1e-6)
        clipped, norm = student.clip_gradients([g], value, eps=0.0)
        torch.testing.assert_close(clipped[0], g / math.sqrt(1000), rtol=1e-6, atol=0)
    zero = torch.zeros(10, device="cuda")
    clipped, norm = student.clip_gradients([zero], 1.0)
    assert float(norm) == 0.0 and not clipped[0].any()
    for bad in (float("inf"), float("nan")):
        p = torch.nn.Parameter(torch.ones(10, device="cuda"))
        q = torch.nn.Parameter(torch.ones(10, device="cuda"))
        p.grad, q.grad = torch.ones(10, device="cuda"), torch.ones(10, device="cuda")
        p.grad[3] = bad
        with pytest.raises(RuntimeError, match="total norm"):
            student.clip_grad_norm_([p, q], 1.0, error_if_nonfinite=True)
        assert torch.equal(q.grad, torch.ones(10, device="cuda"))  # nothing was scaled
        r = [p.grad.clone(), q.grad.clone()]
        mine = student.clip_grad_norm_([p, q], 1.0)
        ps = [torch.nn.Parameter(torch.ones(10, device="cuda")) for _ in r]
        for a, g in zip(ps, r):
            a.grad = g
        theirs = torch.nn.utils.clip_grad_norm_(ps, 1.0)
        torch.testing.assert_close(mine, theirs, equal_nan=True)
        for a, b in zip((p, q), ps):
            torch.testing.assert_close(a.grad, b.grad, equal_nan=True)


def test_clip_refuses_a_gradient_twice():
    p = torch.nn.Parameter(torch.ones(4, device="cuda"))
    p.grad = torch.ones(4, device="cuda")
    with pytest.raises(ValueError, match="twice"):
        student.clip_grad_norm_([p, p], 1.0)
    assert float(student.grad_norm([p.grad, p.grad])) == pytest.approx(math.sqrt(8.0))


def test_clip_in_place_is_a_write_that_autograd_sees():
    p = torch.nn.Parameter(torch.ones(4, device="cuda"))
    p.grad = torch.full((4,), 3.0, device="cuda")
    kept = (p * p.grad).sum()  # saves the gradient
    student.clip_grad_norm_([p], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.backward()


def test_clip_offsets_behind_32_bits():
    g = torch.zeros(2 ** 31 + 77, device="cuda", dtype=BF16)
    g[-1], g[2 ** 31 - 1], g[5] = 3.0, 4.0, 12.0
    clipped, norm = student.clip_gradients([g], 6.5, eps=0.0)
    assert float(norm) == 13.0
    at = torch.tensor([5, 2 ** 31 - 1, 2 ** 31 + 76], device="cuda")
    assert clipped[0][at].tolist() == [6.0, 2.0, 1.5] and int((clipped[0] != 0).sum()) == 3


# ------------------------------------------------------------------------------------------ calls of every kind
def test_offsets_behind_32_bits():
    """Rows, tokens and heads whose element offsets do not fit 32 bits."""
    far = 2 ** 31 + 64
    buf = torch.zeros(far + 4096, device="cuda", dtype=BF16)
    cfg, pos = student.RotaryConfig(64), torch.tensor([[5], [9]], device="cuda")
    q = torch.as_strided(buf, (2, 1, 3, 64), (far, 64, 64, 1))
    small = randn(2, 1, 3, 64, seed=1, dtype=BF16)
    q.copy_(small)
    w = torch.ones(64, device="cuda")
    for a, b in zip(student.qk_norm_rotary(q, q, w, w, pos, cfg), student.qk_norm_rotary(small, small, w, w, pos, cfg)):
        assert torch.equal(a, b)
    for n in (2, 9, 140):  # each kernel of the feed-forward block
        ld = (far // (n - 1) + 8) // 8 * 8
        x = torch.as_strided(torch.zeros(ld * (n - 1) + 64, device="cuda", dtype=BF16), (n, 64), (ld, 1))
        small = randn(n, 64, seed=2, dtype=BF16)
        x.copy_(small)
        _, wg, wu, _ = glu_inputs(1, 64, 72, BF16, 3)
        assert torch.equal(student.gated_linear_unit(x, wg, wu), student.gated_linear_unit(small, wg, wu))


def test_glu_results_behind_32_bits():
    n, h, f = 270_000, 16, 8192
    x, wg, wu = randn(n, h, seed=1, dtype=BF16), randn(f, h, seed=2, dtype=BF16), randn(f, h, seed=3, dtype=BF16)
    leaf = x.detach().requires_grad_(True)
    y = student.gated_linear_unit(leaf, wg, wu, activation="relu")
    dh = torch.zeros_like(y)
    rows = torch.tensor([0, 262_143, 262_144, n - 1], device="cuda")
    dh[rows] = randn(4, f, seed=4, dtype=BF16)
    (dx,) = torch.autograd.grad(y, leaf, dh)
    want = glu64(x[rows], wg, wu, "relu", dh[rows])
    within(y[rows], *want["h"], "h")
    within(dx[rows], *want["dx"], "dx")
    dx[rows] = 0
    assert not dx.any()


def test_second_derivatives_are_refused():
    x, wg, wu, _ = glu_inputs(6, 16, 24, FP32, 5)
    q, w = randn(6, 2, 16, seed=6), torch.ones(16, device="cuda")
    pos, cfg = torch.arange(6, device="cuda"), student.RotaryConfig(16)
    for leaf, call in ((x, lambda t: student.gated_linear_unit(t, wg, wu)),
                       (q, lambda t: student.rotary_embedding(t, t, pos, cfg)[0]),
                       (q, lambda t: student.qk_norm_rotary(t, t, w, w, pos, cfg)[0])):
        leaf = leaf.detach().requires_grad_(True)
        (g,) = torch.autograd.grad(call(leaf).square().sum(), leaf, create_graph=True)
        (plain,) = torch.autograd.grad(call(leaf).square().sum(), leaf)
        assert torch.equal(g, plain)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.sum().backward()


def test_backward_twice_and_kept_graph():
    x, wg, wu, dh = glu_inputs(40, 64, 72, BF16, 7)
    leaf = x.detach().requires_grad_(True)
    y = student.gated_linear_unit(leaf, wg, wu)
    first = torch.autograd.grad(y, leaf, dh, retain_graph=True)[0]
    assert torch.equal(first, torch.autograd.grad(y, leaf, dh)[0])
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, leaf, dh)


def test_mixed_types_inference_mode_and_single_sizes():
    x, wg, wu, _ = glu_inputs(12, 64, 72, BF16, 8)
    want = student.gated_linear_unit(x, wg, wu)
    with torch.inference_mode():
        assert torch.equal(student.gated_linear_unit(x.float(), wg, wu.float()), want)  # bf16 wins
    leaf = x.float().requires_grad_(True)
    student.gated_linear_unit(leaf, wg, wu).sum().backward()
    assert leaf.grad.dtype == FP32
    # dimensions of one element may have any stride
    one = torch.as_strided(x, (1, 64), (7, 1))
    assert torch.equal(student.gated_linear_unit(one, wg, wu), want[:1])
    q = torch.as_strided(randn(1, 5, 1, 64, seed=9, dtype=BF16), (1, 5, 1, 64), (3, 64, 1, 1))
    check_rotary(q, q, torch.arange(5, device="cuda"), student.RotaryConfig(64))


def test_calls_from_several_threads():
    import threading

    x, wg, wu, dh = glu_inputs(40, 64, 72, BF16, 10)
    grads = [randn(500, seed=i) for i in range(120)]
    want = student.gated_linear_unit(x, wg, wu)
    want_clip, want_norm = student.clip_gradients(grads, 1.0)
    torch.cuda.synchronize()
    wrong = []

    def work(k):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(30):
                leaf = x.detach().requires_grad_(True)
                y = student.gated_linear_unit(leaf, wg, wu)
                torch.autograd.grad(y, leaf, dh)
                clipped, norm = student.clip_gradients(grads, 1.0)
            stream.synchronize()
        if not (torch.equal(y, want) and torch.equal(norm, want_norm)
                and all(torch.equal(a, b) for a, b in zip(clipped, want_clip))):
            wrong.append(k)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


# ------------------------------------------------------------------------------------------ together, streams, graphs
def _step(x, gate, up, wq, wk, qkv, pos, cfg):
    """Forward, backward and clipping of the operators in a row, as a student's layer would run them."""
    n = x.shape[0]
    q, k = student.qk_norm_rotary(qkv[:, :256].view(n, 4, 64), qkv[:, 256:384].view(n, 2, 64), wq, wk, pos, cfg)
    q, k = student.rotary_embedding(q, k, pos, cfg)
    h = student.gated_linear_unit(x + q.flatten(1) + k.flatten(1).repeat(1, 2), gate, up)
    grads = torch.autograd.grad((h * h).sum(), (x, gate, up, wq, wk, qkv))
    clipped, norm = student.clip_gradients(grads, 1.0)
    return [h.detach(), norm, *clipped]


def _step_inputs(n, seed):
    ins = [randn(n, 256, seed=seed, dtype=BF16), randn(320, 256, seed=seed + 1, dtype=BF16, scale=0.06),
           randn(320, 256, seed=seed + 2, dtype=BF16, scale=0.06), 1 + randn(64, seed=seed + 3, scale=0.1),
           1 + randn(64, seed=seed + 4, scale=0.1), randn(n, 512, seed=seed + 5, dtype=BF16)]
    return [t.requires_grad_(True) for t in ins], torch.arange(n, device="cuda") * 3, student.RotaryConfig(64)


@pytest.mark.parametrize("n", [20, 300])
def test_step_is_the_same_on_every_run_and_stream(n):
    leaves, pos, cfg = _step_inputs(n, 100)
    want = _step(*leaves, pos, cfg)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(4):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(_step(*leaves, pos, cfg))
    torch.cuda.synchronize()
    for run in got:
        for a, b in zip(run, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("n", [20, 300])
def test_step_replays_from_two_graphs(n):
    leaves, pos, cfg = _step_inputs(n, 200)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            _step(*leaves, pos, cfg)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    captured = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _step(*leaves, pos, cfg)
        captured.append((g, out))
    fresh, _, _ = _step_inputs(n, 300)
    with torch.no_grad():
        for a, b in zip(leaves, fresh):
            a.copy_(b)
    for g, _ in captured:
        g.replay()
    torch.cuda.synchronize()
    want = _step(*fresh, pos, cfg)
    for _, out in captured:
        for a, b in zip(out, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("which", ["glu", "rotary", "norm"])
@pytest.mark.parametrize("accumulate", [False, True])
def test_captured_backward_is_refused_while_an_eager_graph_of_its_leaves_lives(which, accumulate):
    x, wg, wu, _ = glu_inputs(20, 64, 72, BF16, 12)
    q, w = randn(6, 2, 16, seed=13), torch.ones(16, device="cuda")
    pos, cfg = torch.arange(6, device="cuda"), student.RotaryConfig(16)
    call = {"glu": lambda t: student.gated_linear_unit(x, t, wu),
            "rotary": lambda t: student.rotary_embedding(t, q, pos, cfg)[0],
            "norm": lambda t: student.qk_norm_rotary(q, t, w, w, pos, cfg)[1]}[which]
    leaf = (wg if which == "glu" else q).detach().requires_grad_(True)

    def step():
        y = call(leaf)
        dy = torch.ones_like(y)
        if accumulate:
            y.backward(dy)
            return leaf.grad
        return torch.autograd.grad(y, leaf, dy)[0]

    want = step().clone()
    leaf.grad = None
    eager = call(leaf)  # recorded on the default stream
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="still lives"):
        with torch.cuda.graph(graph):
            step()
    del eager, graph
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        eager = call(leaf)  # a graph of another stream does no harm
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(2):
        if accumulate:
            got.zero_()
        graph.replay()
        assert torch.equal(got, want)
    del eager


def test_operators_and_loss_in_one_step():
    """A student's block, the distillation loss on its output and clipping: every gradient against the
    same step in 64 bits."""
    import orda_ce_kernel as ok

    n, d, f, v = 96, 64, 96, 200
    dt = BF16
    x, gate, up, _ = glu_inputs(n, d, f, dt, 400)
    qkv, wq, wk = randn(n, 3 * 64, seed=404, dtype=dt), 1 + randn(32, seed=405, scale=0.1), 1 + randn(32, seed=406, scale=0.1)
    head = randn(v, f, seed=407, dtype=dt, scale=0.1)
    teacher = randn(n, f, seed=408, dtype=dt)
    labels = torch.randint(0, v, (n,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    labels[::9] = -100
    pos, cfg = torch.arange(n, device="cuda"), student.RotaryConfig(32)
    leaves = [t.detach().requires_grad_(True) for t in (x, qkv, wq, wk, gate, up, head)]
    x_, qkv_, wq_, wk_, gate_, up_, head_ = leaves
    q, k = student.qk_norm_rotary(qkv_[:, :64].view(n, 2, 32), qkv_[:, 64:128].view(n, 2, 32), wq_, wk_, pos, cfg)
    hidden = student.gated_linear_unit(x_ + q.flatten(1) * k.flatten(1), gate_, up_)
    loss = ok.distillation_loss(hidden, head_, labels, ok.TiedTeacher(teacher), teacher_ce_weight=0.0, kl_weight=0.5).loss
    loss.backward()

    ref = [t.detach().double().requires_grad_(True) for t in (x, qkv, wq, wk, gate, up, head)]

    def norm_turn(t, w):
        z = t * (t.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w
        a, b = z[..., :16], z[..., 16:]
        ang = pos.double()[:, None, None] * torch.tensor(cfg.frequencies(), device="cuda", dtype=torch.float64)
        return torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1)

    rq, rk = norm_turn(ref[1][:, :64].view(n, 2, 32), ref[2]), norm_turn(ref[1][:, 64:128].view(n, 2, 32), ref[3])
    r_in = ref[0] + rq.flatten(1) * rk.flatten(1)
    r_h = torch.nn.functional.silu(r_in @ ref[4].T) * (r_in @ ref[5].T)
    z, zt = r_h @ ref[6].T, teacher.double() @ ref[6].detach().T
    keep = labels != -100
    ce = torch.nn.functional.cross_entropy(z[keep], labels[keep])
    kl = (zt.softmax(-1) * (zt.log_softmax(-1) - z.log_softmax(-1))).sum(-1)[keep].mean()
    (ce + 0.5 * kl).backward()
    assert float(loss) == pytest.approx(float(ce + 0.5 * kl), rel=1e-2)
    for name, a, b in zip(("x", "qkv", "wq", "wk", "gate", "up", "head"), leaves, ref):
        # six chained steps that each round to bf16 (2^-9 rms each): 2.5% of the tensor's norm at the outside
        rel = float((a.grad.double() - b.grad).norm() / b.grad.norm())
        assert rel < 2.5e-2, (name, rel)
    grads = [t.grad for t in leaves]
    norm, factor = clip64(grads, 0.1)
    want = [g.double() * factor for g in grads]
    assert float(student.clip_grad_norm_(leaves, 0.1)) == pytest.approx(norm, rel=2.0 ** -22)
    for t, w in zip(leaves, want):
        within(t.grad, w, w.abs() * (half(t.dtype) + 2.0 ** -22))


@pytest.mark.parametrize("qk_norm", [False, True])
def test_training_benchmark_model_through_the_operators(qk_norm):
    """The training benchmark's decoder with its rotations, norms and feed-forward blocks through the
    operators, against the same weights through plain PyTorch in 64 bits."""
    from orda_ce_kernel.benchmarks.train_step import TinyLM

    cfg = dict(dim=256, q_heads=4, kv_heads=2, n_layers=2, ffn_dim=704)
    torch.manual_seed(3)
    plain = TinyLM(500, cfg, 64, qk_norm).cuda().double()
    fused = TinyLM(500, cfg, 64, qk_norm, ops=True).cuda()
    fused.load_state_dict(plain.state_dict())  # fp32 copies of the same weights
    ids = torch.randint(0, 500, (2, 48), device="cuda")
    dy = randn(2, 48, 256, seed=9)
    for lm in (plain, fused):
        (lm.hidden(ids) * dy.to(lm.embed.weight.dtype)).sum().backward()
    for (name, a), (_, b) in zip(fused.named_parameters(), plain.named_parameters()):
        # fp32 against fp64 through two layers: sums of up to 704 terms at 2^-24 each step
        rel = float((a.grad.double() - b.grad).norm() / b.grad.norm())
        assert rel < 1e-4, (name, rel)


def test_training_benchmark_step_clips_through_the_operators():
    from orda_ce_kernel.benchmarks import train_step

    step = train_step.make_step("orda_b200-ops", "separate-student", 32_768, 128, "cuda", qk_norm=True, clip_norm=0.5)
    first, second = float(step()), float(step())
    assert math.isfinite(first) and math.isfinite(second) and first != second


@pytest.mark.parametrize("act", ["silu"])
def test_compiled_calls_match_eager(act):
    x, gate, up, dh = glu_inputs(40, 66, 75, BF16, 500)
    q, k = randn(2, 20, 4, 64, seed=501, dtype=BF16), randn(2, 20, 2, 64, seed=502, dtype=BF16)
    w = [1 + randn(64, seed=503 + i, scale=0.1) for i in range(2)]
    pos, cfg = torch.arange(20, device="cuda"), student.RotaryConfig(64, scaling="linear", factor=2.0)

    def fn(x, gate, up, q, k, wq, wk):
        h = student.gated_linear_unit(x, gate, up, activation=act)
        a, b = student.qk_norm_rotary(q, k, wq, wk, pos, cfg)
        c, d = student.rotary_embedding(a, b, pos, cfg)
        return h, c, d

    results = []
    for f in (fn, torch.compile(fn, fullgraph=True)):
        leaves = [t.detach().clone().requires_grad_(True) for t in (x, gate, up, q, k, *w)]
        out = f(*leaves)
        sum((o.float() * o.float()).sum() for o in out).backward()
        results.append([*out, *[t.grad for t in leaves]])
    for a, b in zip(*results):
        assert torch.equal(a, b)
