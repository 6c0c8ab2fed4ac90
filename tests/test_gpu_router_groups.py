"""Group-limited routing (ttamd_router_topk_grouped, the grouped gate + route
entry points) and the gradient of the routing weights, against a plain
restatement in 64 bits.

Picks are whole numbers and must be equal: both sides select on 64-bit
scores.  Scores are 64-bit values rounded once to fp32, at most half a step
(2^-24) plus the kernel's own exponential (below 1e-14), so 2^-23 bounds them.
The gradient is fp32 arithmetic on at most E terms; its bound is stated where
it is checked."""
from __future__ import annotations

import importlib

import numpy as np
import pytest
import torch

from gpu_util import DEV, announce, bf16_dev, rand_bf16, to_np

EPS = 1e-20


def plain(z, K, func, norm, scale, bias, G, kept, value):
    """The definition, in numpy float64: NaN first, then values descending, ties to the lower id."""
    z = np.asarray(z, np.float64)
    T, E = z.shape
    with np.errstate(all="ignore"):
        if func == "softmax":
            m = np.fmax.reduce(z, axis=1, keepdims=True)
            ex = np.exp(z - m)
            p = ex / ex.sum(1, keepdims=True)
        else:
            p = 1.0 / (1.0 + np.exp(-z))
        v = p if bias is None else p + np.asarray(bias, np.float64)

        def order(a):  # indices in the selection's order, along the last axis
            key = np.where(np.isnan(a), np.inf, np.where(np.isposinf(a), 1e300, a))
            return np.argsort(-key, axis=-1, kind="stable")

        top = np.take_along_axis(v.reshape(T, G, E // G), order(v.reshape(T, G, E // G)), 2)
        gv = top[:, :, :2].sum(2) if value == "top2" else top[:, :, 0]
    keep = order(gv)[:, :kept]
    idx = np.empty((T, K), np.int64)
    for t in range(T):
        ids = np.concatenate([np.arange(g * (E // G), (g + 1) * (E // G)) for g in sorted(keep[t])])
        idx[t] = ids[order(v[t, ids])[:K]]
    w = np.take_along_axis(p, idx, 1)
    s = w / (w.sum(1, keepdims=True) + EPS) if norm else w
    return p, s * scale, idx


def plain_grad(p, idx, g, func, norm, scale):
    w = np.take_along_axis(p, idx, 1)
    g = np.asarray(g, np.float64) * scale
    if norm:
        S = w.sum(1, keepdims=True) + EPS
        g = g / S - (g * w).sum(1, keepdims=True) / (S * S)
    dp = np.zeros_like(p)
    for k in range(idx.shape[1]):
        np.add.at(dp, (np.arange(len(p)), idx[:, k]), g[:, k])
    return p * (dp - (dp * p).sum(1, keepdims=True)) if func == "softmax" else dp * p * (1 - p)


CASES = [
    # T, E, K, groups, kept, value
    (1, 256, 8, 8, 4, "top2"),
    (33, 256, 8, 8, 4, "top2"),
    (2049, 256, 8, 8, 4, "top2"),      # four tokens per wave
    (4099, 160, 6, 8, 3, "max"),       # 10 experts per lane
    (5, 60, 4, 5, 2, "top2"),          # groups do not fill the lanes
    (3001, 60, 4, 5, 2, "top2"),
    (2500, 240, 16, 3, 2, "top2"),     # too many per lane for 16 lanes
    (70, 64, 1, 64, 1, "top2"),        # groups of one expert
    (70, 64, 16, 64, 16, "max"),
    (2100, 16, 16, 1, 1, "top2"),      # one group: plain top-k of every expert
    (40, 1, 1, 1, 1, "max"),
    (11, 1000, 7, 8, 2, "max"),        # above 256 experts
    (9, 1023, 16, 33, 5, "top2"),
    (2300, 128, 8, 16, 16, "top2"),    # every group kept
    (2300, 9, 3, 9, 4, "top2"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("T,E,K,G,kept,value", CASES)
@pytest.mark.parametrize("func", ["sigmoid", "softmax"])
def test_grouped_topk_matches_plain(ops, T, E, K, G, kept, value, func):
    rng = np.random.default_rng(T * 7 + E)
    for bf16, with_bias, norm in ((False, True, True), (True, False, False), (True, True, False)):
        z = rng.standard_normal((T, E)).astype(np.float32) * 1.5
        zt = torch.from_numpy(z).to(DEV)
        if bf16:  # many exact ties
            zt = zt.to(torch.bfloat16)
            z = to_np(zt)
        bias = (rng.standard_normal(E) * 0.05).astype(np.float32) if with_bias else None
        bt = None if bias is None else torch.from_numpy(bias).to(DEV)
        announce(f"grouped topk T={T} E={E} K={K} G={G} kept={kept} {value} {func} bf16={bf16} bias={with_bias}")
        s, i = ops.router_topk(zt, K, func, norm, 2.5, bt, EPS, num_groups=G, topk_groups=kept, group_score=value)
        torch.cuda.synchronize()
        _, ws, wi = plain(z, K, func, norm, 2.5, bias, G, kept, value)
        np.testing.assert_array_equal(i.cpu().numpy(), wi)
        np.testing.assert_allclose(s.cpu().numpy(), ws, rtol=2.0 ** -23, atol=1e-38)


@pytest.mark.gpu
@pytest.mark.parametrize("func", ["sigmoid", "softmax"])
@pytest.mark.parametrize("T", [7, 2061])
def test_grouped_topk_special_values(ops, func, T):
    """Rows of equal logits, of NaN, of -inf and of large ones; biases of
    -inf (a whole group, all experts of a group but one, every expert) and
    +inf."""
    rng = np.random.default_rng(5)
    E, K, G, kept = 32, 5, 8, 2
    z = rng.standard_normal((T, E)).astype(np.float32)
    z[0] = 0.0
    z[1, 3] = np.nan
    z[2] = -np.inf if func == "sigmoid" else -1e30
    z[3] = np.where(np.arange(E) % 3 == 0, -np.inf, z[3])
    z[4] = 30.0 * z[4]
    z[5] = np.where(np.arange(E) % 2 == 0, 1e4, -1e4) if func == "softmax" else 0.25
    inf = np.inf
    biases = [None, np.zeros(E)]
    b = rng.standard_normal(E) * 0.1
    b1 = b.copy(); b1[4:8] = -inf; b1[9:12] = -inf
    b2 = np.full(E, -inf)
    b3 = b.copy(); b3[20] = inf; b3[13] = inf
    b4 = b.copy(); b4[20] = inf; b4[21] = -inf; b4[22] = -inf; b4[23] = -inf
    for n, bias in enumerate(biases + [b1, b2, b3, b4]):
        bt = None if bias is None else torch.from_numpy(bias.astype(np.float32)).to(DEV)
        for value in ("top2", "max"):
            announce(f"grouped topk special values {func} T={T} bias {n} {value}")
            s, i = ops.router_topk(torch.from_numpy(z).to(DEV), K, func, False, 1.0, bt, EPS, num_groups=G,
                                   topk_groups=kept, group_score=value)
            torch.cuda.synchronize()
            _, ws, wi = plain(z, K, func, False, 1.0, None if bias is None else bias.astype(np.float32), G, kept,
                              value)
            np.testing.assert_array_equal(i.cpu().numpy(), wi)
            np.testing.assert_allclose(s.cpu().numpy(), ws, rtol=2.0 ** -23, atol=1e-38)


@pytest.mark.gpu
@pytest.mark.parametrize("func", ["sigmoid", "softmax"])
@pytest.mark.parametrize("T", [7, 2061])
def test_grouped_topk_huge_logits(ops, func, T):
    """Logits whose differences or sizes leave exp's range (their scores are
    equal then: the lower ids win), up to fp32's largest."""
    rng = np.random.default_rng(51)
    E, K, G, kept = 64, 6, 8, 3
    for size in (3e3, 1e10, 1e30, 3.4e38):
        z = (rng.uniform(-1.0, 1.0, (T, E)) * size).astype(np.float32)
        z[:, ::5] = np.float32(0.999 * size)
        announce(f"grouped topk huge logits {func} T={T} {size}")
        s, i = ops.router_topk(torch.from_numpy(z).to(DEV), K, func, True, 1.0, None, EPS, num_groups=G,
                               topk_groups=kept)
        torch.cuda.synchronize()
        _, ws, wi = plain(z, K, func, True, 1.0, None, G, kept, "top2")
        np.testing.assert_array_equal(i.cpu().numpy(), wi)
        np.testing.assert_allclose(s.cpu().numpy(), ws, rtol=2.0 ** -23, atol=1e-38)


@pytest.mark.gpu
def test_grouped_topk_unaligned_and_strided(ops):
    """Logits that start off a 16-byte border, and a column slice."""
    rng = np.random.default_rng(6)
    T, E = 2100, 64
    flat = torch.from_numpy(rng.standard_normal(T * E + 1).astype(np.float32)).to(DEV)
    wide = torch.from_numpy(rng.standard_normal((T, 2 * E)).astype(np.float32)).to(DEV)
    for z in (flat[1:].view(T, E), wide[:, 3:3 + E]):
        s, i = ops.router_topk(z, 6, "sigmoid", True, 1.0, num_groups=4, topk_groups=2)
        _, ws, wi = plain(to_np(z), 6, "sigmoid", True, 1.0, None, 4, 2, "top2")
        np.testing.assert_array_equal(i.cpu().numpy(), wi)
        np.testing.assert_allclose(s.cpu().numpy(), ws, rtol=2.0 ** -23)
    s, i = ops.router_topk(wide[:0], 6, "sigmoid", num_groups=4, topk_groups=2)
    assert s.shape == (0, 6) and i.shape == (0, 6)


@pytest.mark.gpu
@pytest.mark.parametrize("T,E,K,G,kept,value", [c for c in CASES if c[1] > 1])
@pytest.mark.parametrize("func,norm", [("sigmoid", True), ("softmax", False), ("softmax", True)])
def test_topk_backward_matches_plain(ops, T, E, K, G, kept, value, func, norm):
    """Each fp32 term is within a few 2^-24 of its size; the terms of one
    element sum to at most |g|_1 (1 + 1/S) in size (scores are at most 1), and
    the softmax dot and the sums over K add at most E roundings.  For K = 1
    with renormalisation the terms cancel to zero, so the bound is absolute."""
    rng = np.random.default_rng(T + 3 * E)
    for bf16 in (False, True):
        zt = torch.from_numpy(rng.standard_normal((T, E)).astype(np.float32) * 1.5).to(DEV)
        zt = zt.to(torch.bfloat16) if bf16 else zt
        g = torch.from_numpy(rng.standard_normal((T, K)).astype(np.float32)).to(DEV)
        announce(f"topk backward T={T} E={E} K={K} {func} norm={norm} bf16={bf16}")
        _, i = ops.router_topk(zt, K, func, norm, 2.5, num_groups=G, topk_groups=kept, group_score=value)
        dz = ops.router_topk_backward(g, i, zt, func, norm, 2.5, EPS)
        torch.cuda.synchronize()
        assert dz.dtype == zt.dtype
        p, _, _ = plain(to_np(zt), K, func, norm, 2.5, None, G, kept, value)
        idx = i.cpu().numpy()
        ref = plain_grad(p, idx, to_np(g), func, norm, 2.5)
        w = np.take_along_axis(p, idx, 1)
        size = 2.5 * np.abs(to_np(g)).sum(1, keepdims=True) * (2 / w.sum(1, keepdims=True) if norm else 1.0)
        tol = size * p * (E + 16) * 2.0 ** -23 + (np.abs(ref) * 2.0 ** -8 if bf16 else 0.0) + 1e-38
        assert (np.abs(to_np(dz) - ref) <= tol).all()


@pytest.mark.gpu
def test_topk_backward_same_index_twice_and_out_of_range(ops):
    rng = np.random.default_rng(8)
    T, E, K = 37, 48, 4
    z = rng.standard_normal((T, E)).astype(np.float32)
    idx = rng.integers(0, E, (T, K))
    idx[:, 1] = idx[:, 0]
    g = rng.standard_normal((T, K)).astype(np.float32)
    dev = lambda a: torch.from_numpy(a).to(DEV)  # noqa: E731
    for func in ("sigmoid", "softmax"):
        p, _, _ = plain(z, K, func, False, 1.0, None, 1, 1, "max")
        dz = ops.router_topk_backward(dev(g), dev(idx), dev(z), func)
        np.testing.assert_allclose(to_np(dz), plain_grad(p, idx, g, func, False, 1.0), atol=2e-5)
        bad = idx.copy()
        bad[:, 3] = np.where(np.arange(T) % 2 == 0, -1, E + 5)
        dz = ops.router_topk_backward(dev(g), dev(bad), dev(z), func)
        np.testing.assert_allclose(to_np(dz), plain_grad(p, idx[:, :3], g[:, :3], func, False, 1.0), atol=2e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("func,norm", [("sigmoid", True), ("softmax", False)])
def test_topk_autograd_matches_differences(func, norm):
    """functional.router_topk's gradient against central differences of the
    plain 64-bit scores (the picks fixed): the difference quotient's own error
    is about h^2 = 1e-8 of third derivatives below 2.5 |g|."""
    F = importlib.import_module("torchtitan-ascend_amd.functional")
    rng = np.random.default_rng(10)
    T, E, K, G, kept = 5, 24, 4, 6, 2
    z = rng.standard_normal((T, E)).astype(np.float32)
    g = rng.standard_normal((T, K))
    zt = torch.from_numpy(z).to(DEV).requires_grad_(True)
    s, i = F.router_topk(zt, K, func, norm, 2.5, num_groups=G, topk_groups=kept)
    assert not i.requires_grad
    s.backward(torch.from_numpy(g.astype(np.float32)).to(DEV))
    idx = i.cpu().numpy()

    def loss(zz):
        p, _, _ = plain(zz, K, func, norm, 2.5, None, G, kept, "top2")
        w = np.take_along_axis(p, idx, 1)
        w = w / (w.sum(1, keepdims=True) + EPS) if norm else w
        return float((2.5 * w * g).sum())

    h = 1e-4
    for t, e in [(0, int(idx[0, 0])), (1, int(idx[1, 2])), (2, 0), (4, 23), (3, int(idx[3, 3]))]:
        d = np.zeros_like(z, dtype=np.float64)
        d[t, e] = h
        num = (loss(z + d) - loss(z - d)) / (2 * h)
        assert abs(num - float(zt.grad[t, e])) < 2e-6 * (1 + abs(num)) * 10


@pytest.mark.gpu
@pytest.mark.parametrize("T,D,E,K,G,kept,func,norm", [
    (1, 256, 16, 2, 4, 2, "sigmoid", True),
    (50, 2048, 256, 8, 8, 4, "sigmoid", True),
    (4111, 512, 256, 8, 8, 4, "softmax", False),
    (2500, 256, 60, 4, 5, 2, "sigmoid", False),
])
def test_grouped_router_and_route(ops, T, D, E, K, G, kept, func, norm):
    """router_fused and router_route with groups: the picks of the plain
    selection on the bf16 logits that router_fused returns, and the counts and
    stable order of those picks."""
    rng = np.random.default_rng(T + D)
    x, w = bf16_dev(rand_bf16(rng, (T, D))), bf16_dev(rand_bf16(rng, (E, D), 0.05))
    bias = torch.from_numpy((rng.standard_normal(E) * 0.05).astype(np.float32)).to(DEV)
    how = dict(num_groups=G, topk_groups=kept)
    announce(f"grouped router T={T} D={D} E={E} K={K} G={G}")
    s, i, lg = ops.router_fused(x, w, K, func, norm, 2.5, bias, return_logits=True, **how)
    _, _, lg0 = ops.router_fused(x, w, K, func, norm, 2.5, bias, return_logits=True)
    assert torch.equal(lg, lg0)
    _, ws, wi = plain(to_np(lg), K, func, norm, 2.5, to_np(bias), G, kept, "top2")
    np.testing.assert_array_equal(i.cpu().numpy(), wi)
    np.testing.assert_allclose(s.cpu().numpy(), ws, rtol=2.0 ** -23)
    seen = torch.ones(E, device=DEV)
    s2, i2, r = ops.router_route(x, w, K, func, norm, 2.5, bias, tokens_per_expert=seen, **how)
    torch.cuda.synchronize()
    assert torch.equal(s2, s) and torch.equal(i2, i)
    flat = wi.reshape(-1)
    np.testing.assert_array_equal(r.counts.cpu().numpy(), np.bincount(flat, minlength=E))
    np.testing.assert_array_equal(r.sorted_indices.cpu().numpy(), np.argsort(flat, kind="stable"))
    np.testing.assert_array_equal(to_np(seen), 1 + np.bincount(flat, minlength=E))


@pytest.mark.gpu
def test_grouped_router_backward_follows_the_picks(ops):
    """functional.router with groups: the gradients are router_backward's for its own picks."""
    F = importlib.import_module("torchtitan-ascend_amd.functional")
    rng = np.random.default_rng(12)
    T, D, E, K = 600, 256, 64, 6
    x, w = bf16_dev(rand_bf16(rng, (T, D))), bf16_dev(rand_bf16(rng, (E, D), 0.05))
    g = torch.from_numpy(rng.standard_normal((T, K)).astype(np.float32)).to(DEV)
    xg, wg = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    s, i = F.router(xg, wg, K, "sigmoid", True, 2.5, num_groups=8, topk_groups=3, group_score="max")
    s.backward(g)
    _, i2, lg = ops.router_fused(x, w, K, "sigmoid", True, 2.5, return_logits=True, num_groups=8, topk_groups=3,
                                 group_score="max")
    assert torch.equal(i, i2)
    dx, dw = ops.router_backward(g, i2, lg, x, w, "sigmoid", True, 2.5, dw_dtype=torch.bfloat16)
    assert torch.equal(xg.grad, dx) and torch.equal(wg.grad, dw)


@pytest.mark.gpu
def test_grouped_topk_captured(ops):
    """Captured and replayed on new logits: every replay equals the eager call."""
    rng = np.random.default_rng(13)
    T, E, K = 300, 256, 8
    z = torch.empty(T, E, device=DEV)
    g = torch.ones(T, K, device=DEV)
    how = dict(num_groups=8, topk_groups=4)
    ops.router_topk(z.zero_(), K, "sigmoid", **how)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s, i = ops.router_topk(z, K, "sigmoid", True, **how)
        dz = ops.router_topk_backward(g, i, z, "sigmoid", True)
    for _ in range(3):
        z.copy_(torch.from_numpy(rng.standard_normal((T, E)).astype(np.float32)))
        graph.replay()
        s2, i2 = ops.router_topk(z, K, "sigmoid", True, **how)
        dz2 = ops.router_topk_backward(g, i2, z, "sigmoid", True)
        torch.cuda.synchronize()
        assert torch.equal(s, s2) and torch.equal(i, i2) and torch.equal(dz, dz2)


# ---------------------------------------------------------------------------
# Refusals (CPU: nothing is launched)
# ---------------------------------------------------------------------------
_lib = importlib.import_module("torchtitan-ascend_amd._lib")


def _topk(E=64, K=4, G=8, kept=2, value=0, T=4, func=1):
    import ctypes

    p = ctypes.c_void_p(256)
    rc = _lib.load().ttamd_router_topk_grouped(p, 0, None, T, E, K, G, kept, value, func, 0, 0.0, 1.0, p, p, None)
    assert rc == 1
    return _lib.load().ttamd_last_error().decode()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_router_backward_without_tokens(ops, dtype):
    """No tokens: the gate weight's gradient is zeros, whatever memory it gets."""
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=DEV)  # noqa: E731
    announce("router backward without tokens")
    for _ in range(3):
        torch.full((8, 256), float("nan"), dtype=dtype, device=DEV)  # what the allocator hands out next
        dx, dw = ops.router_backward(torch.zeros(0, 2, device=DEV), torch.zeros(0, 2, dtype=torch.int64, device=DEV),
                                     bf(0, 8), bf(0, 256), bf(8, 256), dw_dtype=dtype)
        assert dx.shape == (0, 256) and dw.shape == (8, 256) and not dw.any()


@pytest.mark.gpu
def test_grouped_topk_past_32_bits(ops):
    """More than 2^31 logits: the last tokens are those of a small call."""
    T, E, K, few = 9_000_001, 256, 8, 500
    z = torch.empty(T, E, dtype=torch.bfloat16, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(6)
    z[: T - few].fill_(0.25)
    z[T - few:] = torch.randn(few, E, device=DEV, generator=g)
    announce("grouped top-k past 32 bits")
    for func in ("sigmoid", "softmax"):
        how = dict(score_func=func, route_norm=True, num_groups=8, topk_groups=4)
        s, i = ops.router_topk(z, K, **how)
        ss, si = ops.router_topk(z[T - few:], K, **how)
        assert torch.equal(i[T - few:], si) and torch.equal(s[T - few:], ss)
        assert torch.equal(i[: T - few], i[:1].expand(T - few, K))
        d = ops.router_topk_backward(s, i, z, func, True)
        assert torch.equal(d[T - few:], ops.router_topk_backward(ss, si, z[T - few:], func, True))
        del s, i, d


def test_grouped_topk_refusals():
    assert "divide num_experts" in _topk(G=7)
    assert "num_groups" in _topk(E=128, G=128)
    assert "num_groups" in _topk(G=0)
    assert "topk_groups" in _topk(kept=9)
    assert "topk_groups" in _topk(kept=0)
    assert "topk must be" in _topk(K=16, kept=1)   # 8 experts in the kept group
    assert "topk must be" in _topk(K=17, kept=8)
    assert "topk must be" in _topk(K=0)
    assert "group_score" in _topk(value=2)
    assert "score_func" in _topk(func=2)
    assert "num_experts" in _topk(E=2048, G=8, kept=8)
    assert "num_tokens" in _topk(T=-1)
    assert "num_tokens" in _topk(T=(1 << 24) + 1)


def test_grouped_arguments_come_together(ops):
    with pytest.raises(ValueError, match="together"):
        ops._groups(8, None, "top2")
    with pytest.raises(ValueError, match="together"):
        ops._groups(None, 2, "top2")
    with pytest.raises(ValueError, match="group_score"):
        ops._groups(8, 2, "mean")
    assert ops._groups(None, None, "top2") is None
    assert ops._groups(8, 2, "max") == (8, 2, 1)


def test_grouped_ops_need_a_gpu(ops):
    z = torch.zeros(4, 64)
    with pytest.raises(RuntimeError, match="HIP device"):
        ops.router_topk(z, 4, num_groups=8, topk_groups=2)
    with pytest.raises(RuntimeError, match="HIP device"):
        ops.router_topk_backward(torch.zeros(4, 4), torch.zeros(4, 4, dtype=torch.int64), z)


# ---------------------------------------------------------------------------
# The 64-bit arithmetic's own bounds
# ---------------------------------------------------------------------------
def grad_bound(p, idx, ref, g, func, norm, scale, bf16):
    """What topk_backward_kernel may be off by.  Its scores are within 2^-43 of
    themselves (exponential and sum 2^-45.6 each, reciprocal 2^-45) and
    everything else is 64-bit, so an element is within a few such steps (16:
    2^-39) of the sum of its terms' sizes, before any cancels; then one
    rounding to fp32, or two to bf16, and half a step of the smallest numbers."""
    w = np.take_along_axis(p, idx, 1)
    d = np.abs(np.asarray(g, np.float64)) * scale
    if norm:
        S = w.sum(1, keepdims=True) + EPS
        d = d / S + (d * w).sum(1, keepdims=True) / (S * S)
    a = np.zeros_like(p)
    for k in range(idx.shape[1]):
        np.add.at(a, (np.arange(len(p)), idx[:, k]), d[:, k])
    size = p * (a + (d * w).sum(1, keepdims=True)) if func == "softmax" else p * a
    step = 2.0 ** -8 + 2.0 ** -23 if bf16 else 2.0 ** -24
    return np.abs(ref) * step + size * 2.0 ** -39 + (2.0 ** -133 if bf16 else 2.0 ** -149)


@pytest.mark.gpu
@pytest.mark.parametrize("T,E,K,G,kept,value", [(4099, 160, 6, 8, 3, "max"), (33, 256, 8, 8, 4, "top2"),
                                                (70, 64, 1, 64, 1, "top2"), (9, 1023, 16, 33, 5, "top2"),
                                                (50, 48, 2, 4, 2, "top2")])
@pytest.mark.parametrize("func,norm", [("sigmoid", True), ("sigmoid", False), ("softmax", False), ("softmax", True)])
@pytest.mark.parametrize("peak", [0.0, 10.0, 20.0])
def test_topk_backward_is_64_bit(ops, T, E, K, G, kept, value, func, norm, peak):
    """Ordinary rows and peaked ones (a logit 10 or 20 above the rest), where a
    renormalised weight or a softmax score is close to 1 and the differences
    of the formulas cancel."""
    rng = np.random.default_rng(T + 5 * E + int(peak))
    z = rng.standard_normal((T, E)).astype(np.float32) * 1.5
    z[np.arange(T), rng.integers(0, E, T)] += np.float32(peak)
    for bf16 in (False, True):
        zt = torch.from_numpy(z).to(DEV)
        zt = zt.to(torch.bfloat16) if bf16 else zt
        g = rng.standard_normal((T, K)).astype(np.float32)
        announce(f"64-bit topk backward T={T} E={E} K={K} {func} norm={norm} peak={peak} bf16={bf16}")
        _, i = ops.router_topk(zt, K, func, norm, 2.5, num_groups=G, topk_groups=kept, group_score=value)
        dz = ops.router_topk_backward(torch.from_numpy(g).to(DEV), i, zt, func, norm, 2.5, EPS)
        torch.cuda.synchronize()
        p, _, _ = plain(to_np(zt), K, func, norm, 2.5, None, G, kept, value)
        idx = i.cpu().numpy()
        ref = plain_grad(p, idx, g, func, norm, 2.5)
        tol = grad_bound(p, idx, ref, g, func, norm, 2.5, bf16)
        got = dz.cpu().double().numpy()
        assert (np.abs(got - ref) <= tol).all(), float((np.abs(got - ref) / tol).max())


def truncated(v):
    """The first 42 places of the values."""
    return (np.asarray(v, np.float64).view(np.uint64) & ~np.uint64(1023)).view(np.float64)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [7, 2061])
@pytest.mark.parametrize("G,kept,value", [(1, 1, "max"), (4, 4, "top2"), (4, 2, "max"), (4, 2, "top2")])
def test_saturated_sigmoids_compare_42_places(ops, T, G, kept, value):
    """Sigmoid scores so close to 1 that 64 bits still tell them apart and 42
    places do not (logits of 30 and 36): equal values, so the lower id (group)
    wins.  None of these logits' scores is within the kernel's 2^-45 of a
    border of the 42 places."""
    rng = np.random.default_rng(T + G)
    E, K = 32, 6
    pool = np.array([28.0, 28.5, 29.0, 29.5, 30.0, 30.5, 31.0, 32.0, 33.0, 35.0, 36.0, 38.0, 40.0])
    z = rng.choice(pool, (T, E)).astype(np.float32)
    announce(f"saturated sigmoids T={T} G={G} kept={kept} {value}")
    s, i = ops.router_topk(torch.from_numpy(z).to(DEV), K, "sigmoid", False, 1.0, num_groups=G, topk_groups=kept,
                           group_score=value)
    torch.cuda.synchronize()
    score = 1.0 / (1.0 + np.exp(-z.astype(np.float64)))
    v = truncated(score)
    best = -np.sort(-v.reshape(T, G, E // G), axis=2)
    gv = truncated(best[:, :, 0] + best[:, :, 1]) if value == "top2" else best[:, :, 0]
    keep = np.argsort(-gv, axis=1, kind="stable")[:, :kept]
    in_kept = np.zeros((T, G), bool)
    np.put_along_axis(in_kept, keep, True, 1)
    v = np.where(np.repeat(in_kept, E // G, axis=1), v, -1.0)
    want = np.argsort(-v, axis=1, kind="stable")[:, :K]
    np.testing.assert_array_equal(i.cpu().numpy(), want)
    np.testing.assert_allclose(s.cpu().numpy(), np.take_along_axis(score, want, 1), rtol=2.0 ** -23)
    # what the documentation says of it: the definition's own 64-bit order differs here
    assert (np.argsort(-np.where(v < 0, -1.0, score), axis=1, kind="stable")[:, :K] != want).any()
