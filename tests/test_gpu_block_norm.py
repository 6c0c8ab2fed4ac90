"""The norms before and after a block with gate, residual scale and combine
(ttamd_residual_norm and its backward) against their definition in 64 bits
(gradients by torch's autograd in float64).

Bounds, per element, derived before the first run.  u and n are rounded once:
half a step of their type (2^-8 bf16, 2^-24 fp32) of the value.  Before that,
fp32 arithmetic: u is a sum of terms whose sizes add up to S = |residual| +
scale |act p|; each factor (the mean square's sum over D, the root, the
products, exp) adds at most 2^-20 relative for D <= 8192 (D / 64 sequential
additions per lane at 2^-24 each, random signs, and a dozen more).  n divides
by a root of the same relative error.  Gradients sum the same way; their term
sizes are computed in 64 bits beside the values."""
from __future__ import annotations

import importlib

import numpy as np
import pytest
import torch

from gpu_util import DEV, announce

EPS = 1e-6
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
F32 = 2.0 ** -19


def case(rng, T, D, stream="bf16", weights="bf16", gate="none", post=True, pre=True, residual=True, K=0,
         gathered=False, scored=False):
    dt = {"bf16": torch.bfloat16, "fp32": torch.float32}
    mk = lambda *s, t, m=0.0, sd=1.0: torch.from_numpy(rng.standard_normal(s) * sd + m).to(dt[t]).to(DEV)  # noqa: E731
    c = dict(residual=mk(T, D, t=stream, sd=3.0) if residual else None,
             post_weight=mk(D, t=weights, m=1.0, sd=0.2) if post else None,
             pre_weight=mk(D, t=weights, m=1.0, sd=0.2) if pre else None)
    shape = {"none": None, "token": (T, 1), "channel": (1, D), "full": (T, D)}[gate]
    c["gate"] = None if shape is None else mk(*shape, t=weights)
    c["branch"] = mk(T * max(K, 1), D, t="bf16")
    c["inverse"] = torch.from_numpy(rng.permutation(T * K).astype(np.int32)).to(DEV) if gathered else None
    c["probs"] = torch.from_numpy(rng.random((T, K)).astype(np.float32)).to(DEV) if scored else None
    return c


def wide(c):
    return {k: c[k].double().requires_grad_(True) for k in ("branch", "residual", "post_weight", "gate", "pre_weight")
            if c[k] is not None}


def define(w, func, scale, T, K=0, inverse=None, probs=None):
    f = w["branch"]
    if K:
        order = torch.arange(T * K, device=f.device) if inverse is None else inverse.long()
        p = torch.ones(T * K, 1, device=f.device) if probs is None else probs.double().reshape(-1, 1)
        f = (f[order] * p).view(T, K, -1).sum(1)
    p = f
    if "post_weight" in w:
        p = f / torch.sqrt(f.square().mean(1, keepdim=True) + EPS) * w["post_weight"]
    b = p
    if "gate" in w:
        b = b * (torch.sigmoid(w["gate"]) if func == "sigmoid" else w["gate"])
    b = b * scale
    u = b + w["residual"] if "residual" in w else b
    size = b.detach().abs() + (w["residual"].detach().abs() if "residual" in w else 0.0)
    n = None
    if "pre_weight" in w:
        n = u / torch.sqrt(u.square().mean(1, keepdim=True) + EPS) * w["pre_weight"]
    return u, n, size


def near(got, ref, size, what):
    """|got - ref| <= half a step of the type on the value, plus the fp32 bound on the terms' sizes."""
    d = (got.double() - ref).abs()
    tol = HALF[got.dtype] * (ref.abs() + F32 * size) + F32 * size + 1e-38
    bad = d > tol
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((d / tol).max()):.2f} x"


SHAPES = [
    # T, D
    (1, 8), (3, 64), (1, 2048), (2055, 512), (2100, 1000), (2070, 2048), (33, 2056), (5, 7168), (600, 5120),
    (2, 8192), (2200, 264),
]
FORMS = [
    # stream, weights, gate, func, post, pre, residual, scale
    ("bf16", "bf16", "none", "identity", True, True, True, 1.0),
    ("fp32", "fp32", "token", "sigmoid", True, True, True, 0.5),
    ("bf16", "fp32", "channel", "sigmoid", True, True, True, 0.22),
    ("fp32", "bf16", "full", "identity", True, False, True, 1.0),
    ("bf16", "bf16", "full", "sigmoid", False, True, True, 2.0),
    ("bf16", "bf16", "channel", "identity", False, True, False, 1.0),
    ("bf16", "bf16", "token", "identity", True, False, False, -1.0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("T,D", SHAPES)
@pytest.mark.parametrize("form", range(len(FORMS)))
def test_forward(ops, T, D, form):
    stream, weights, gate, func, post, pre, residual, scale = FORMS[form]
    rng = np.random.default_rng(T + D + form)
    c = case(rng, T, D, stream, weights, gate, post, pre, residual)
    announce(f"residual_norm T={T} D={D} {FORMS[form]}")
    u, n = ops.residual_norm(c["branch"], c["residual"], c["post_weight"], c["gate"], func, scale, c["pre_weight"],
                             EPS)
    torch.cuda.synchronize()
    with torch.no_grad():
        ru, rn, size = define(wide(c), func, scale, T)
        assert u.dtype == (c["residual"].dtype if residual else torch.bfloat16)
        near(u, ru, size, "u")
        if pre:
            grow = c["pre_weight"].double().abs() / torch.sqrt(ru.square().mean(1, keepdim=True) + EPS)
            near(n, rn, size * grow, "n")
        else:
            assert n is None


@pytest.mark.gpu
@pytest.mark.parametrize("T,D,K,gathered,scored", [
    (1, 64, 8, True, True), (64, 2048, 8, False, False), (2500, 2048, 8, True, True), (2300, 512, 3, True, False),
    (40, 7168, 6, False, True), (2300, 1032, 2, False, False), (7, 2048, 1, True, True), (5, 8, 64, True, True),
])
@pytest.mark.parametrize("stream", ["bf16", "fp32"])
def test_combine(ops, T, D, K, gathered, scored, stream):
    """The K products and additions of the combine add K 2^-24 of the sum of their sizes, which is at most
    sum_k p |row| in size: folded into the size of p."""
    rng = np.random.default_rng(T + D + K)
    c = case(rng, T, D, stream, "bf16", "token", K=K, gathered=gathered, scored=scored)
    announce(f"combine_norm T={T} D={D} K={K} gathered={gathered} scored={scored} {stream}")
    u, n = ops.combine_norm(c["branch"], K, c["inverse"], c["probs"], c["residual"], c["post_weight"], c["gate"],
                            "sigmoid", 0.7, c["pre_weight"], EPS)
    torch.cuda.synchronize()
    with torch.no_grad():
        w = wide(c)
        ru, rn, size = define(w, "sigmoid", 0.7, T, K, c["inverse"], c["probs"])
        order = torch.arange(T * K, device=DEV) if c["inverse"] is None else c["inverse"].long()
        p = torch.ones(T * K, 1, device=DEV) if c["probs"] is None else c["probs"].double().reshape(-1, 1)
        terms = (w["branch"].abs()[order] * p).view(T, K, D).sum(1)
        f = (w["branch"][order] * p).view(T, K, D).sum(1)
        size = size + terms / torch.sqrt(f.square().mean(1, keepdim=True) + EPS) * w["post_weight"].abs() * 0.7
        near(u, ru, size, "u")
        near(n, rn, size * w["pre_weight"].abs() / torch.sqrt(ru.square().mean(1, keepdim=True) + EPS), "n")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,D", [(1, 8), (2100, 2048), (9, 8192), (2050, 72)])
def test_rms_norm(ops, T, D, dtype):
    rng = np.random.default_rng(T)
    x = torch.from_numpy(rng.standard_normal((T, D)) * 2).to(dtype).to(DEV)
    w = torch.from_numpy(rng.standard_normal(D)).to(torch.float32).to(DEV)
    announce(f"rms_norm T={T} D={D} {dtype}")
    n = ops.rms_norm(x, w, EPS)
    ref = x.double() / torch.sqrt(x.double().square().mean(1, keepdim=True) + EPS) * w.double()
    near(n, ref, ref.abs(), "n")


def term_sizes(w, func, scale, du, dn):
    """Sizes of the terms that each gradient sums, in 64 bits (no cancellation), by the formulas."""
    f, D = w["branch"], w["branch"].shape[1]
    r_f = 1 / torch.sqrt(f.square().mean(1, keepdim=True) + EPS)
    wp = w.get("post_weight", torch.ones(D, device=f.device, dtype=torch.float64))
    p = (f * r_f * wp if "post_weight" in w else f)
    raw = w.get("gate", torch.ones(1, 1, device=f.device, dtype=torch.float64))
    a = torch.sigmoid(raw) if func == "sigmoid" and "gate" in w else raw
    da = a * (1 - a) if func == "sigmoid" else torch.ones_like(a)
    u = scale * a * p + (w["residual"] if "residual" in w else 0.0)
    usize = (scale * a * p).abs() + (w["residual"].abs() if "residual" in w else 0.0)
    r_u = 1 / torch.sqrt(u.square().mean(1, keepdim=True) + EPS)
    g = du.abs()
    out = {}
    if dn is not None:
        q = (dn * w["pre_weight"]).abs()
        g = g + r_u * (q + usize * r_u * (q * usize * r_u).mean(1, keepdim=True))
        out["pre_weight"] = (dn.abs() * usize * r_u).sum(0)
    out["residual"] = g
    gate = abs(scale) * g * p.abs() * da.abs()
    if "gate" in w:
        if w["gate"].shape[1] == 1 and D > 1:
            gate = gate.sum(1, keepdim=True)
        elif w["gate"].shape[0] == 1:
            gate = gate.sum(0, keepdim=True)
        out["gate"] = gate
    dp = abs(scale) * a.abs() * g
    if "post_weight" in w:
        fh = (f * r_f).abs()
        out["post_weight"] = (dp * fh).sum(0)
        q = dp * wp.abs()
        dp = r_f * (q + fh * (q * fh).mean(1, keepdim=True))
    out["branch"] = dp
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("T,D", [(1, 8), (5, 64), (1500, 1000), (300, 2048), (2055, 512), (70, 5120), (9, 7168),
                                 (3, 8192), (1030, 4104)])
@pytest.mark.parametrize("form", range(len(FORMS)))
def test_backward(ops, T, D, form):
    stream, weights, gate, func, post, pre, residual, scale = FORMS[form]
    rng = np.random.default_rng(3 * T + D + form)
    c = case(rng, T, D, stream, weights, gate, post, pre, residual)
    st = c["residual"].dtype if residual else torch.bfloat16
    du = torch.from_numpy(rng.standard_normal((T, D))).to(st).to(DEV)
    dn = torch.from_numpy(rng.standard_normal((T, D))).to(torch.bfloat16).to(DEV) if pre else None
    how = dict(residual=c["residual"], post_weight=c["post_weight"], gate=c["gate"], gate_func=func,
               residual_scale=scale, pre_weight=c["pre_weight"], eps=EPS)
    announce(f"residual_norm backward T={T} D={D} {FORMS[form]}")
    _, _, stats = ops.residual_norm(c["branch"], save_stats=True, **how)
    got = ops.residual_norm_backward(du, dn, c["branch"], stats, **how)._asdict()
    torch.cuda.synchronize()
    w = wide(c)
    u, n, _ = define(w, func, scale, T)
    outs, gs = ([u], [du.double()]) if n is None else ([u, n], [du.double(), dn.double()])
    ref = dict(zip(w, torch.autograd.grad(outs, list(w.values()), gs)))
    with torch.no_grad():
        size = term_sizes({k: v.detach() for k, v in w.items()}, func, scale, du.double(),
                          None if dn is None else dn.double())
    for k in ("branch", "residual", "post_weight", "gate", "pre_weight"):
        if c[k] is None:
            assert got[k] is None
            continue
        assert got[k].dtype == c[k].dtype and got[k].shape == c[k].shape
        near(got[k], ref[k], size[k], f"d{k}")


@pytest.mark.gpu
def test_backward_without_one_of_the_upstream_gradients(ops):
    rng = np.random.default_rng(4)
    T, D = 50, 256
    c = case(rng, T, D, gate="token")
    how = {k: c[k] for k in ("residual", "post_weight", "gate", "pre_weight")}
    _, _, stats = ops.residual_norm(c["branch"], save_stats=True, **how)
    g = torch.from_numpy(rng.standard_normal((T, D))).to(torch.bfloat16).to(DEV)
    zero = torch.zeros_like(g)
    for a, b in ((ops.residual_norm_backward(g, None, c["branch"], stats, **how),
                  ops.residual_norm_backward(g, zero, c["branch"], stats, **how)),
                 (ops.residual_norm_backward(None, g, c["branch"], stats, **how),
                  ops.residual_norm_backward(zero, g, c["branch"], stats, **how))):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


@pytest.mark.gpu
def test_autograd_and_differences(ops):
    """functional.residual_norm and rms_norm deliver the op's gradients through
    autograd, for leaves of both types, and agree with central differences of
    the 64-bit definition along random directions: the loss is a sum of T D
    products of size about 1, its gradient along a direction is off by the
    bf16 rounding of the gradients, 2^-8 of sum |grad direction|."""
    F = importlib.import_module("torchtitan-ascend_amd.functional")
    rng = np.random.default_rng(5)
    T, D = 40, 128
    c = case(rng, T, D, "fp32", "fp32", "token")
    leaves = {k: c[k].clone().requires_grad_(True) for k in ("branch", "residual", "post_weight", "gate", "pre_weight")}
    u, n = F.residual_norm(leaves["branch"], leaves["residual"], leaves["post_weight"], leaves["gate"], "sigmoid", 0.5,
                           leaves["pre_weight"], EPS)
    wu = torch.from_numpy(rng.standard_normal((T, D)).astype(np.float32)).to(DEV)
    wn = torch.from_numpy(rng.standard_normal((T, D))).to(torch.bfloat16).to(DEV)
    ((u * wu).sum() + (n * wn).float().sum()).backward()
    how = dict(residual=c["residual"], post_weight=c["post_weight"], gate=c["gate"], gate_func="sigmoid",
               residual_scale=0.5, pre_weight=c["pre_weight"])
    _, _, stats = ops.residual_norm(c["branch"], save_stats=True, eps=EPS, **how)
    want = ops.residual_norm_backward(wu, wn, c["branch"], stats, **how)
    for k, g in want._asdict().items():
        assert torch.equal(leaves[k].grad, g), k

    def loss(w):
        u, n, _ = define(w, "sigmoid", 0.5, T)
        return float((u * wu.double()).sum() + (n * wn.double()).sum())

    h = 1e-5
    for k in leaves:
        d = torch.from_numpy(rng.standard_normal(tuple(c[k].shape))).to(DEV)
        with torch.no_grad():
            hi, lo = wide(c), wide(c)
            hi[k] = hi[k] + h * d
            lo[k] = lo[k] - h * d
            num = (loss(hi) - loss(lo)) / (2 * h)
        terms = leaves[k].grad.double() * d
        assert abs(num - float(terms.sum())) <= 2.0 ** -8 * float(terms.abs().sum()) + 1e-4 * (1 + abs(num))
    # only one of the outputs used, rms_norm, and no gradient at all
    x = c["residual"].clone().requires_grad_(True)
    wt = c["pre_weight"].clone().requires_grad_(True)
    y = F.rms_norm(x.view(4, 10, D), wt, EPS)
    assert y.shape == (4, 10, D) and y.dtype == torch.bfloat16
    y.backward(wn.view(4, 10, D))
    _, st = ops.rms_norm(c["residual"], c["pre_weight"], EPS, True)
    ref = ops.residual_norm_backward(None, wn, None, st, residual=c["residual"], pre_weight=c["pre_weight"])
    assert torch.equal(x.grad, ref.residual) and torch.equal(wt.grad, ref.pre_weight)
    assert ref.branch is None and ref.gate is None
    u, n = F.residual_norm(c["branch"])
    assert n is None and not u.requires_grad


@pytest.mark.gpu
def test_rms_norm_backward_matches_definition(ops):
    rng = np.random.default_rng(15)
    for T, D, dt in ((1, 64, torch.float32), (700, 2048, torch.bfloat16), (33, 8192, torch.float32)):
        x = torch.from_numpy(rng.standard_normal((T, D))).to(dt).to(DEV)
        w = torch.from_numpy(rng.standard_normal(D).astype(np.float32)).to(DEV)
        g = torch.from_numpy(rng.standard_normal((T, D))).to(torch.bfloat16).to(DEV)
        announce(f"rms_norm backward T={T} D={D} {dt}")
        _, st = ops.rms_norm(x, w, EPS, True)
        got = ops.residual_norm_backward(None, g, None, st, residual=x, pre_weight=w)
        xd, wd = x.double().requires_grad_(True), w.double().requires_grad_(True)
        n = xd / torch.sqrt(xd.square().mean(1, keepdim=True) + EPS) * wd
        rx, rw = torch.autograd.grad(n, [xd, wd], g.double())
        with torch.no_grad():
            r = 1 / torch.sqrt(xd.square().mean(1, keepdim=True) + EPS)
            q, xh = (g.double() * wd).abs(), (xd * r).abs()
            near(got.residual, rx, r * (q + xh * (q * xh).mean(1, keepdim=True)), "dx")
            near(got.pre_weight, rw, (g.double().abs() * xh).sum(0), "dw")


@pytest.mark.gpu
def test_special_rows_stay_in_their_row(ops):
    """A row of zeros (the root of eps alone), of infinities and of NaN: other
    rows are untouched, and the rows give what the definition gives."""
    rng = np.random.default_rng(6)
    for T, D in ((8, 512), (2200, 512), (8, 5120)):
        c = case(rng, T, D)
        c["branch"][1] = 0
        c["residual"][1] = 0
        clean = ops.residual_norm(c["branch"], c["residual"], c["post_weight"], pre_weight=c["pre_weight"])
        assert not clean[1][1].any() and not clean[0][1].any()
        bad = c["branch"].clone()
        bad[3, 5] = float("nan")
        bad[5, 7] = float("inf")
        u, n = ops.residual_norm(bad, c["residual"], c["post_weight"], pre_weight=c["pre_weight"])
        keep = torch.ones(T, dtype=torch.bool, device=DEV)
        keep[3] = keep[5] = False
        assert torch.equal(u[keep], clean[0][keep]) and torch.equal(n[keep], clean[1][keep])
        assert bool(u[3].isnan().all()) and bool(n[3].isnan().all())
        assert bool(n[5].isnan().all())  # inf * 0


@pytest.mark.gpu
def test_empty_strided_and_other_stream(ops):
    rng = np.random.default_rng(7)
    c = case(rng, 0, 64)
    u, n, st = ops.residual_norm(c["branch"], c["residual"], c["post_weight"], pre_weight=c["pre_weight"],
                                 save_stats=True)
    assert u.shape == (0, 64) and n.shape == (0, 64)
    g = ops.residual_norm_backward(u, n, c["branch"], st, residual=c["residual"], post_weight=c["post_weight"],
                                   pre_weight=c["pre_weight"])
    assert not g.post_weight.any() and not g.pre_weight.any() and g.branch.shape == (0, 64)
    # column slices of wider tensors, and a transposed one
    wide_b = torch.randn(40, 200, device=DEV).to(torch.bfloat16)
    wide_r = torch.randn(128, 40, device=DEV).t()
    w = torch.ones(128, device=DEV)
    a = ops.residual_norm(wide_b[:, 8:136], wide_r, w, pre_weight=w)
    b = ops.residual_norm(wide_b[:, 8:136].contiguous(), wide_r.contiguous(), w, pre_weight=w)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s = ops.residual_norm(wide_b[:, 8:136], wide_r, w, pre_weight=w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(s[1], a[1])


@pytest.mark.gpu
def test_captured_forward_and_backward(ops):
    """Forward and backward in one graph, replayed on new inputs with eager
    work between: every replay equals the eager calls."""
    rng = np.random.default_rng(8)
    T, D = 700, 1024
    c = case(rng, T, D, gate="channel")
    g = torch.randn(T, D, device=DEV).to(torch.bfloat16)
    how = dict(residual=c["residual"], post_weight=c["post_weight"], gate=c["gate"], pre_weight=c["pre_weight"])

    def step():
        u, n, st = ops.residual_norm(c["branch"], save_stats=True, **how)
        return (u, n, *ops.residual_norm_backward(g, g, c["branch"], st, **how))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        c["branch"].normal_()
        g.normal_()
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


# ---------------------------------------------------------------------------
# Refusals (CPU: nothing is launched)
# ---------------------------------------------------------------------------
def _forward(rows=256, inverse=None, probs=None, T=4, D=64, K=1, residual=256, post=None, gate=None, kind=0, pre=256,
             eps=1e-6, mask=0, u=256, n=256):
    import ctypes

    L = importlib.import_module("torchtitan-ascend_amd._lib")
    p = lambda v: None if v is None else ctypes.c_void_p(v)  # noqa: E731
    rc = L.load().ttamd_residual_norm(p(rows), p(inverse), p(probs), T, D, K, p(residual), p(post), p(gate), kind, 0,
                                      1.0, p(pre), eps, mask, p(u), p(n), None, None)
    assert rc == 1
    return L.load().ttamd_last_error().decode()


@pytest.mark.gpu
def test_output_in_place_of_the_residual(ops):
    """u_out may be the residual itself (the C entry point)."""
    from importlib import import_module

    lib = import_module("torchtitan-ascend_amd._lib")
    rng = np.random.default_rng(41)
    for stream in ("bf16", "fp32"):
        c = case(rng, 5000, 520, stream=stream)
        want, _ = ops.residual_norm(c["branch"], c["residual"], c["post_weight"], pre_weight=c["pre_weight"], eps=EPS)
        res = c["residual"].clone()
        n = torch.empty_like(c["branch"])
        announce(f"u over the {stream} residual")
        p = lambda t: t.data_ptr()  # noqa: E731
        lib.call("ttamd_residual_norm", p(c["branch"]), None, None, 5000, 520, 1, p(res), p(c["post_weight"]), None, 0, 0,
                 1.0, p(c["pre_weight"]), EPS, 1 if stream == "fp32" else 0, p(res), p(n), None,
                 torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(res, want)


@pytest.mark.gpu
def test_backward_without_rows(ops):
    """No tokens: the weights' and the channel gate's gradients are zeros."""
    rng = np.random.default_rng(42)
    c = case(rng, 3, 264, gate="channel")
    stats = torch.empty(2, 0, device=DEV)
    announce("backward without rows")
    for _ in range(3):
        torch.full((1 << 16,), float("nan"), device=DEV)  # what the allocator hands out next
        g = ops.residual_norm_backward(c["branch"][:0], c["branch"][:0], c["branch"][:0], stats, c["residual"][:0],
                                       c["post_weight"], c["gate"], "sigmoid", 0.5, c["pre_weight"])
        assert g.branch.shape == (0, 264) and g.residual.shape == (0, 264)
        for t, like in ((g.post_weight, c["post_weight"]), (g.gate, c["gate"]), (g.pre_weight, c["pre_weight"])):
            assert t.shape == like.shape and not t.any()


@pytest.mark.gpu
def test_rows_past_32_bits(ops):
    """More than 2^31 elements: the last rows are those of a small call."""
    T, D, few = 300_000, 8192, 257
    g = torch.Generator(device=DEV).manual_seed(5)
    mk = lambda *s: torch.randn(*s, device=DEV, generator=g, dtype=torch.bfloat16)  # noqa: E731
    branch, residual, w1, w2 = mk(T, D), mk(T, D), mk(D), mk(D)
    announce("rows past 32 bits")
    u, n, st = ops.residual_norm(branch, residual, w1, pre_weight=w2, eps=EPS, save_stats=True)
    tail = slice(T - few, T)
    us, ns, sts = ops.residual_norm(branch[tail], residual[tail], w1, pre_weight=w2, eps=EPS, save_stats=True)
    assert torch.equal(u[tail], us) and torch.equal(n[tail], ns) and torch.equal(st[:, tail], sts)
    got = ops.residual_norm_backward(u, n, branch, st, residual, w1, pre_weight=w2)
    few_grads = ops.residual_norm_backward(us, ns, branch[tail], sts.contiguous(), residual[tail], w1, pre_weight=w2)
    assert torch.equal(got.branch[tail], few_grads.branch) and torch.equal(got.residual[tail], few_grads.residual)
    del u, n, got
    K = 4
    idx = (T - 1 - torch.arange(few * K, device=DEV, dtype=torch.int32)) % T
    every = torch.arange(T, device=DEV, dtype=torch.int32)
    every[: few * K] = idx  # the first tokens read the last rows
    u, _ = ops.combine_norm(branch, K, inverse=every, post_weight=w1, eps=EPS)
    want, _ = ops.combine_norm(branch[idx.long()], K, post_weight=w1, eps=EPS)
    assert torch.equal(u[:few], want)


@pytest.mark.gpu
def test_combine_norm_has_no_backward(ops):
    rows = torch.zeros(8, 64, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    with pytest.raises(RuntimeError, match="no backward"):
        ops.combine_norm(rows, 2)
    with torch.no_grad():
        assert not ops.combine_norm(rows, 2)[0].any()


def test_forward_refusals():
    assert "multiple of 8" in _forward(D=60)
    assert "multiple of 8" in _forward(D=0)
    assert "8192" in _forward(D=8200)
    assert "topk" in _forward(K=65)
    assert "topk" in _forward(K=0)
    assert "num_tokens" in _forward(T=-1)
    assert "num_tokens" in _forward(T=1 << 27, K=4)
    assert "gate" in _forward(kind=2)
    assert "gate" in _forward(gate=256)
    assert "gate_kind" in _forward(gate=256, kind=4)
    assert "f32_mask" in _forward(mask=16)
    assert "both null" in _forward(rows=None, residual=None)
    assert "need rows" in _forward(rows=None, post=256)
    assert "need rows" in _forward(rows=None, inverse=256)
    assert "go together" in _forward(pre=None)
    assert "go together" in _forward(n=None)
    assert "no output" in _forward(u=None, n=None, pre=None)
    assert "aligned" in _forward(rows=258)
    assert "aligned" in _forward(u=264)
    assert "eps" in _forward(eps=-1.0)
    assert "eps" in _forward(eps=float("nan"))


def _backward(branch=256, T=4, D=64, residual=256, post=None, pre=None, rstd=256, dn=None, gp=None, gw=None, ws=256,
              ws_bytes=1 << 30, du=256):
    import ctypes

    L = importlib.import_module("torchtitan-ascend_amd._lib")
    p = lambda v: None if v is None else ctypes.c_void_p(v)  # noqa: E731
    rc = L.load().ttamd_residual_norm_backward(p(du), p(dn), p(branch), T, D, p(residual), p(post), None, 0, 0, 1.0,
                                               p(pre), p(rstd), 0, p(256), p(256), p(gp), None, p(gw), p(ws), ws_bytes,
                                               None)
    assert rc == 1
    return L.load().ttamd_last_error().decode()


def test_backward_refusals():
    assert "rstd" in _backward(rstd=None)
    assert "dn needs" in _backward(dn=256)
    assert "not given" in _backward(gp=256)
    assert "not given" in _backward(gw=256)
    assert "workspace" in _backward(ws=None)
    assert "workspace" in _backward(ws_bytes=64)
    assert "aligned" in _backward(du=260)
    L = importlib.import_module("torchtitan-ascend_amd._lib").load()
    sizes = [L.ttamd_residual_norm_backward_workspace_bytes(t, 512) for t in (0, 1, 2, 100, 1000, 5000, 10 ** 6)]
    assert sizes == sorted(sizes) and sizes[0] == 0


def test_python_refusals(ops):
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="HIP device"):
        ops.residual_norm(x, x)
    with pytest.raises(RuntimeError, match="HIP device"):
        ops.rms_norm(x, x[0])
    with pytest.raises(RuntimeError, match="HIP device"):
        ops.combine_norm(x, 2)
    dev = x.device
    bad = [(dict(residual=x[:2]), "residual"), (dict(post_weight=x[0, :8]), "post_weight"),
           (dict(pre_weight=x), "pre_weight"), (dict(gate=x[:, 0]), "gate"), (dict(gate=x[:3]), "gate"),
           (dict(gate_func="tanh"), "gate_func")]
    base = dict(residual=None, post_weight=None, gate=None, gate_func="identity", pre_weight=None)
    for change, word in bad:
        with pytest.raises(ValueError, match=word):
            ops._norm_operands(dev, 4, 64, **{**base, **change})
    with pytest.raises(TypeError, match="residual"):
        ops._norm_operands(dev, 4, 64, **{**base, "residual": x.half()})
    assert ops._norm_operands(dev, 4, 64, **{**base, "gate": x[:, :1].float()})[3] == 1
    assert ops._norm_operands(dev, 4, 64, **{**base, "gate": x[:1]})[3] == 2
    assert ops._norm_operands(dev, 4, 64, **{**base, "gate": x})[3] == 3
    assert ops._norm_operands(dev, 1, 64, **{**base, "gate": x[:1]})[3] == 2
    assert ops._norm_operands(dev, 1, 64, **{**base, "gate": x[:1, :1]})[3] == 1


def test_backward_refuses_a_missing_channel_gate_without_tokens():
    """post_weight's gradient is written without tokens too, and a channel gate
    is a factor of it: without the gate nothing is launched."""
    import ctypes

    L = importlib.import_module("torchtitan-ascend_amd._lib").load()
    p = ctypes.c_void_p(256)
    rc = L.ttamd_residual_norm_backward(None, None, p, 0, 64, None, p, None, 2, 0, 1.0, None, p, 0, p, None, p, None,
                                        None, None, 0, None)
    assert rc == 1
    assert "gate" in L.ttamd_last_error().decode()
