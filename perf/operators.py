"""Operators of a distillation training step around the loss, and of its student's token-by-token run.

* ``glu``    - ``gated_linear_unit``: ``h = act(x Wg^T) * (x Wu^T)``; training cases add its gradients.
* ``rotary`` - ``rotary_embedding``: positions rotated into queries and keys.
* ``qknorm`` - ``qk_norm_rotary``: per-head RMS norms of queries and keys, rotated in the same pass.
* ``clip``   - ``clip_gradients``: the global norm over many gradients, and the clipped gradients.

``run`` computes them in plain torch operations, or, with ``own`` set, through
``orda_ce_kernel.student``.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------ cases
def _glu(name, rows, hidden, ffn, dtype, act, train):
    return {"name": name, "op": "glu", "rows": rows, "hidden": hidden, "ffn": ffn, "dtype": dtype, "act": act,
            "train": train}


def _rot(name, op, batch, seq, q_heads, kv_heads, head_dim, rotary_dim, layout, scaling, factor, far, dtype, train):
    return {"name": name, "op": op, "batch": batch, "seq": seq, "q_heads": q_heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "rotary_dim": rotary_dim, "layout": layout, "scaling": scaling, "factor": factor,
            "far": far, "dtype": dtype, "train": train}


def _clip(name, layers, dim, ffn, vocab, dtype, max_norm):
    return {"name": name, "op": "clip", "layers": layers, "dim": dim, "ffn": ffn, "vocab": vocab, "dtype": dtype,
            "max_norm": max_norm}


def listed():
    return [
        # one token of one sequence through a wide student's feed-forward block: reads the weights once
        _glu("glu 1 row 4096", 1, 4096, 11264, "bf16", "silu", False),
        # a batch of sequences that each decode one token, benchmark student's sizes, GeGLU
        _glu("glu 37 rows 1024", 37, 1024, 2816, "fp16", "gelu_tanh", False),
        # training step of the benchmark's student: 16 sequences of 512 tokens
        _glu("glu train 1024", 8192, 1024, 2816, "bf16", "silu", True),
        # the same block at the width of the 4096-wide lm_head workload
        _glu("glu train 4096", 8192, 4096, 11264, "bf16", "silu", True),
        # packed batch whose sizes fit no tile and no 16-byte row
        _glu("glu train ragged", 1111, 1000, 2730, "fp16", "gelu", True),
        # one new token for each of 64 sequences, far positions, context stretched eightfold
        _rot("rotary decode", "rotary", 64, 1, 32, 8, 128, 128, "half", "yarn", 8.0, 1000000, "bf16", False),
        # training batch of the benchmark's student, half of each head rotated, neighbouring pairs
        _rot("rotary train partial", "rotary", 16, 2048, 8, 2, 128, 64, "interleaved", "none", 1.0, 0, "bf16", True),
        # a few tokens of the benchmark's student
        _rot("qk norm decode", "qknorm", 7, 1, 8, 2, 128, 128, "half", "none", 1.0, 30000, "fp16", False),
        # training batch of a 4096-wide student with 8 key heads
        _rot("qk norm train", "qknorm", 8, 2048, 32, 8, 128, 128, "half", "linear", 4.0, 0, "bf16", True),
        # gradients of a tiny student with odd sizes, fp32: launches and the host decide
        _clip("clip small fp32", 2, 130, 355, 1009, "fp32", 1.0),
        # the benchmark's student: 8 layers and a 32768-row embedding
        _clip("clip student", 8, 1024, 2816, 32768, "bf16", 1.0),
        # a 4096-wide student of 4 layers and its 128256-row lm_head
        _clip("clip large", 4, 4096, 11264, 128256, "bf16", 1.0),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["glu", "rotary", "qknorm", "clip"])
    if op == "glu":
        train = rng.random() < 0.5
        hidden = _spread(rng, 200, 4096)
        hidden = hidden if rng.random() < 0.3 else max(8, hidden // 8 * 8)
        ffn = int(hidden * rng.uniform(1.5, 2.75))
        ffn = ffn if rng.random() < 0.3 else ffn // 8 * 8
        return _without_name(_glu("", _spread(rng, 64, 8192) if train else _spread(rng, 1, 8192), hidden, ffn,
                                  rng.choice(["bf16", "fp16"]), rng.choice(["silu", "gelu", "gelu_tanh", "relu"]), train))
    if op in ("rotary", "qknorm"):
        train = rng.random() < 0.5
        head_dim = rng.choice([64, 80, 96, 128, 128, 256, 50])
        rotary_dim = rng.choice([head_dim, head_dim, head_dim // 4 * 2])
        kv = rng.choice([1, 2, 4, 8])
        scaling = rng.choice(["none", "linear", "ntk", "yarn"])
        return _without_name(_rot("", op, rng.randint(1, 16), _spread(rng, 16, 1024) if train else rng.randint(1, 4),
                                  kv * rng.choice([1, 3, 4, 8][: 2 if kv == 8 else 4]), kv, head_dim, rotary_dim,
                                  rng.choice(["half", "interleaved"]), scaling,
                                  1.0 if scaling == "none" else float(rng.choice([2, 4, 8, 32])),
                                  rng.choice([0, 4000, 120000, 1000000]), rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                                  train))
    dim = _spread(rng, 60, 2048)
    return _without_name(_clip("", rng.randint(1, 8), dim, int(dim * rng.uniform(1.5, 2.75)), _spread(rng, 500, 100000),
                               rng.choice(["bf16", "fp16", "fp32"]), rng.choice([0.1, 1.0, 1000000.0])))


def _without_name(case):
    return {k: v for k, v in case.items() if k != "name"}


# ------------------------------------------------------------------------------------------ inputs
def _clip_shapes(case):
    """Parameter shapes of the training-step student: per layer two norms, qkv, proj, gate, up, down."""
    d, f = case["dim"], case["ffn"]
    layer = [(d,), (d,), (d + d // 2, d), (d, d), (f, d), (f, d), (d, f)]
    return layer * case["layers"] + [(case["vocab"], d), (d,)]


def _frequencies(case):
    """Angle per position of each rotated pair, 64 bits, and the factor of the rotated values."""
    d, base, s = case["rotary_dim"], 10000.0, case["factor"]
    i = torch.arange(0, d, 2, dtype=torch.float64)
    magnitude = 1.0
    if case["scaling"] == "ntk":
        base *= s ** (d / (d - 2))
    theta = base ** (-i / d)
    if case["scaling"] == "linear":
        theta = theta / s
    elif case["scaling"] == "yarn":
        turns = 4096 * theta / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        theta = theta / s * (1.0 - keep) + theta * keep
        magnitude = 0.1 * math.log(s) + 1.0
    return theta, magnitude


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dt)

    s = {"case": case}
    if case["op"] == "glu":
        n, h, f = case["rows"], case["hidden"], case["ffn"]
        s["x"] = randn(n, h)
        s["gate"] = randn(f, h, scale=h ** -0.5)
        s["up"] = randn(f, h, scale=h ** -0.5)
        if case["train"]:
            s["dh"] = randn(n, f, scale=1e-2)
    elif case["op"] in ("rotary", "qknorm"):
        b, t, hq, hk, d = (case[k] for k in ("batch", "seq", "q_heads", "kv_heads", "head_dim"))
        qkv = randn(b, t, (hq + 2 * hk) * d)  # what the fused projection leaves
        s["q"] = qkv[..., : hq * d].view(b, t, hq, d)
        s["k"] = qkv[..., hq * d: (hq + hk) * d].view(b, t, hk, d)
        first = torch.randint(0, case["far"] + 1, (b, 1), generator=g, device="cuda")
        s["positions"] = first + torch.arange(t, device="cuda")
        if case["op"] == "qknorm":
            s["q_weight"] = 1.0 + randn(d, scale=0.1)
            s["k_weight"] = 1.0 + randn(d, scale=0.1)
        if case["train"]:
            s["dq"], s["dk"] = randn(b, t, hq, d, scale=1e-2), randn(b, t, hk, d, scale=1e-2)
        theta, s["magnitude"] = _frequencies(case)
        s["theta"] = theta.cuda()
    else:
        # gradients are small and differ in size from tensor to tensor
        s["grads"] = [randn(*shape, scale=1e-3 * (1 + i % 3)) for i, shape in enumerate(_clip_shapes(case))]
    if own:
        pkg = os.path.join(os.getcwd(), "orda-knowledge-distillation-kernel_b200")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        from orda_ce_kernel import student

        s["student"] = student
        if case["op"] in ("rotary", "qknorm"):
            s["config"] = student.RotaryConfig(
                head_dim=case["head_dim"], rotary_dim=case["rotary_dim"], base=10000.0, layout=case["layout"],
                scaling=case["scaling"], factor=case["factor"], original_positions=4096)
    return s


# ------------------------------------------------------------------------------------------ plain forms
def _act(act, g):
    """act(g) and its derivative."""
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return g * s, s * (1.0 + g * (1.0 - s))
    if act == "relu":
        on = (g > 0).to(g.dtype)
        return g * on, on
    if act == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    c = math.sqrt(2.0 / math.pi)
    th = torch.tanh(c * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1.0 + th), 0.5 * (1.0 + th) + 0.5 * g * (1.0 - th * th) * c * (1.0 + 3 * 0.044715 * g * g)


def _plain_glu(s):
    case = s["case"]
    dt = s["x"].dtype
    x, wg, wu = s["x"].float(), s["gate"].float(), s["up"].float()
    g, u = x @ wg.T, x @ wu.T
    a, da = _act(case["act"], g)
    h = (a * u).to(dt)
    if not case["train"]:
        return h
    dh = s["dh"].float()
    dg, du = dh * u * da, dh * a
    return {"h": h, "dx": (dg @ wg + du @ wu).to(dt), "d_gate": (dg.T @ x).to(dt), "d_up": (du.T @ x).to(dt)}


def _rotate(x, cos, sin, case):
    """x [B, T, heads, D] in 32 bits, cos / sin [B, T, 1, rotary / 2]; the rest of the head passes."""
    r = case["rotary_dim"]
    if case["layout"] == "half":
        a, b = x[..., : r // 2], x[..., r // 2: r]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    else:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    return torch.cat([turned, x[..., r:]], dim=-1)


def _plain_rotary(s):
    case = s["case"]
    dt = s["q"].dtype
    angle = s["positions"].double()[..., None] * s["theta"]
    cos = (torch.cos(angle) * s["magnitude"]).float()[:, :, None]
    sin = (torch.sin(angle) * s["magnitude"]).float()[:, :, None]
    q, k = s["q"].float(), s["k"].float()
    if case["op"] == "rotary":
        out = {"q": _rotate(q, cos, sin, case).to(dt), "k": _rotate(k, cos, sin, case).to(dt)}
        if case["train"]:
            out["dq"] = _rotate(s["dq"].float(), cos, -sin, case).to(dt)
            out["dk"] = _rotate(s["dk"].float(), cos, -sin, case).to(dt)
        return out
    wq, wk = s["q_weight"].float(), s["k_weight"].float()
    rq = torch.rsqrt((q * q).mean(-1, keepdim=True) + 1e-6)
    rk = torch.rsqrt((k * k).mean(-1, keepdim=True) + 1e-6)
    nq, nk = q * rq, k * rk
    out = {"q": _rotate(nq * wq, cos, sin, case).to(dt), "k": _rotate(nk * wk, cos, sin, case).to(dt)}
    if case["train"]:
        zq, zk = _rotate(s["dq"].float(), cos, -sin, case), _rotate(s["dk"].float(), cos, -sin, case)
        out["dq_weight"] = (zq * nq).sum((0, 1, 2)).to(dt)
        out["dk_weight"] = (zk * nk).sum((0, 1, 2)).to(dt)
        zq, zk = zq * wq, zk * wk
        out["dq"] = (rq * (zq - nq * (zq * nq).mean(-1, keepdim=True))).to(dt)
        out["dk"] = (rk * (zk - nk * (zk * nk).mean(-1, keepdim=True))).to(dt)
    return out


def _plain_clip(s):
    grads = s["grads"]
    norm = torch.sqrt(torch.stack([g.double().square().sum() for g in grads]).sum())
    factor = (s["case"]["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    return {"norm": norm.float(), "grads": [(g.float() * factor).to(g.dtype) for g in grads]}


# ------------------------------------------------------------------------------------------ the framework's calls
def _own_glu(s):
    ops, case = s["student"], s["case"]
    if not case["train"]:
        return ops.gated_linear_unit(s["x"], s["gate"], s["up"], activation=case["act"])
    x, gate, up = (s[k].detach().requires_grad_(True) for k in ("x", "gate", "up"))
    h = ops.gated_linear_unit(x, gate, up, activation=case["act"])
    dx, d_gate, d_up = torch.autograd.grad(h, (x, gate, up), s["dh"])
    return {"h": h.detach(), "dx": dx, "d_gate": d_gate, "d_up": d_up}


def _own_rotary(s):
    ops, case = s["student"], s["case"]
    norm = case["op"] == "qknorm"
    names = ("q", "k", "q_weight", "k_weight") if norm else ("q", "k")
    leaves = [s[n].detach().requires_grad_(True) if case["train"] else s[n] for n in names]
    call = ops.qk_norm_rotary if norm else ops.rotary_embedding
    q, k = call(*leaves, s["positions"], s["config"])
    out = {"q": q.detach(), "k": k.detach()}
    if case["train"]:
        out.update(zip(["d" + n for n in names], torch.autograd.grad((q, k), leaves, (s["dq"], s["dk"]))))
    return out


def _own_clip(s):
    clipped, norm = s["student"].clip_gradients(s["grads"], s["case"]["max_norm"])
    return {"norm": norm, "grads": clipped}


def run(state):
    op = state["case"]["op"]
    if own:
        return _own_glu(state) if op == "glu" else _own_clip(state) if op == "clip" else _own_rotary(state)
    return _plain_glu(state) if op == "glu" else _plain_clip(state) if op == "clip" else _plain_rotary(state)


# ------------------------------------------------------------------------------------------ work
def work(case):
    size = _DTYPES[case["dtype"]].itemsize
    if case["op"] == "glu":
        n, h, f = case["rows"], case["hidden"], case["ffn"]
        inputs, product = n * h + 2 * f * h, 2 * n * h * f
        if not case["train"]:
            return {"bytes": size * (inputs + n * f), "flops": 2 * product}
        # reads x, both weights and dh; writes h and a gradient for each of x and the weights
        return {"bytes": size * (2 * inputs + 2 * n * f), "flops": 6 * product}
    if case["op"] == "clip":
        n = sum(math.prod(shape) for shape in _clip_shapes(case))
        return {"bytes": 2 * size * n, "flops": 3 * n}
    tokens = case["batch"] * case["seq"]
    values = tokens * (case["q_heads"] + case["kv_heads"]) * case["head_dim"]
    norm = case["op"] == "qknorm"
    # forward: q, k in and out; backward: their gradients in and out (and q, k again only for the norms' statistics)
    return {"bytes": size * values * (4 if case["train"] else 2) + 8 * tokens,
            "flops": values * ((20 if norm else 6) if case["train"] else (8 if norm else 3))}


# ------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "glu":
        x, wg, wu = (s[k].double().requires_grad_(True) for k in ("x", "gate", "up"))
        g = torch.einsum("nh,fh->nf", x, wg)
        if case["act"] == "silu":
            a = torch.sigmoid(g) * g
        elif case["act"] == "relu":
            a = torch.where(g > 0, g, torch.zeros_like(g))
        elif case["act"] == "gelu":
            a = 0.5 * g * torch.erfc(-g / math.sqrt(2.0))
        else:  # 0.5 (1 + tanh z) = sigmoid(2 z)
            a = g * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3))
        h = a * torch.einsum("nh,fh->nf", x, wu)
        if not case["train"]:
            return h.detach()
        d = torch.autograd.grad(h, (x, wg, wu), s["dh"].double())
        return {"h": h.detach(), "dx": d[0], "d_gate": d[1], "d_up": d[2]}
    if case["op"] == "clip":
        parts = [torch.linalg.vector_norm(g.double()) for g in s["grads"]]
        norm = torch.linalg.vector_norm(torch.stack(parts))
        factor = min(1.0, case["max_norm"] / (float(norm) + 1e-6))
        return {"norm": norm, "grads": [g.double() * factor for g in s["grads"]]}

    r = case["rotary_dim"]
    theta, magnitude = _frequencies(case)
    phase = torch.polar(torch.tensor(magnitude, dtype=torch.float64).cuda(),
                        s["positions"].double()[..., None, None] * theta.cuda())

    def turn(x):  # each rotated pair as one complex number times magnitude e^(i angle)
        head = x[..., :r]
        pairs = head.unflatten(-1, (r // 2, 2)) if case["layout"] == "interleaved" else head.unflatten(-1, (2, r // 2)).mT
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * phase)
        z = z.flatten(-2) if case["layout"] == "interleaved" else z.mT.flatten(-2)
        return torch.cat([z, x[..., r:]], dim=-1)

    names = ("q", "k", "q_weight", "k_weight") if case["op"] == "qknorm" else ("q", "k")
    leaves = [s[n].double().requires_grad_(True) for n in names]
    if case["op"] == "qknorm":
        y = [turn(x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w) for x, w in zip(leaves[:2], leaves[2:])]
    else:
        y = [turn(x) for x in leaves]
    out = {"q": y[0].detach(), "k": y[1].detach()}
    if case["train"]:
        out.update(zip(["d" + n for n in names], torch.autograd.grad(y, leaves, (s["dq"].double(), s["dk"].double()))))
    return out
