"""The few-token operators and 4-bit weights in the forms beside the plain call: recorded
and replayed, at the ends of the prompt's path, in every kernel that a size may take.

Bounds: test_gpu_decode.py."""
from __future__ import annotations

import importlib
import warnings

import numpy as np
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from gpu_util import DEV, announce
from test_gpu_decode import build, weights

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def decode():
    return importlib.import_module("torchtitan-ascend_amd.decode")


@pytest.fixture(scope="module")
def functional():
    return importlib.import_module("torchtitan-ascend_amd.functional")


def equal(got, want):
    got, want = (v if isinstance(v, tuple) else (v,) for v in (got, want))
    assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))


# ---------------------------------------------------------------------------
# Recordings
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("T", [1, 9, 65])
@pytest.mark.parametrize("bits", [16, 4])
def test_recordings_compute(decode, functional, T, bits):
    """make_fx, torch.jit.trace and torch.compile of the layer on one input, replayed on
    others, give the eager call's bits."""
    rng = np.random.default_rng(T)
    E, K, D, H = 8, 2, 256, 128
    w, _ = build(decode, rng, E, D, H, bits, 128)
    wr, wg = weights(rng, E, D), weights(rng, 1, D)
    proj = decode.pack_e2m1(weights(rng, D, D))

    def step(x):
        h = functional.grouped_mm_e2m1(x, proj)
        return functional.moe_decode(h, wr, *w[:2], K, shared_w13=w[2], shared_w2=w[3], shared_gate=wg)

    x = weights(rng, T, D, scale=1.0)
    announce(f"recordings T={T} bits={bits}")
    with torch.no_grad(), warnings.catch_warnings():
        warnings.simplefilter("ignore")
        forms = [make_fx(step)(x), torch.jit.trace(step, (x,), check_trace=False),
                 torch.compile(step, backend="aot_eager", fullgraph=True)]
        for i in range(3):
            xi = weights(rng, T, D, scale=1.0 + i)
            want = step(xi)
            for f in forms:
                equal(f(xi), want)


@pytest.mark.parametrize("name", ["pack", "pack_matrix", "unpack", "router", "router_gate"])
def test_opcheck_of_weights_and_router(decode, name):
    importlib.import_module("torchtitan-ascend_amd.library")
    rng = np.random.default_rng(1)
    x, wr, wg, w = (weights(rng, *s) for s in ((6, 96), (4, 96), (1, 96), (3, 20, 160)))
    p = decode.pack_e2m1(w)
    ops = torch.ops.ttamd
    op, args = {
        "pack": (ops.pack_e2m1, (w,)),
        "pack_matrix": (ops.pack_e2m1, (w[0].float(),)),
        "unpack": (ops.unpack_e2m1, (p.codes, p.exponents, p.rows, p.cols)),
        "router": (ops.router_decode, (x, wr, 2, "softmax", False, 1.0, None, 1e-20, None, None, "top2", None)),
        "router_gate": (ops.router_decode, (x, wr, 2, "sigmoid", True, 2.5, torch.rand(4, device=DEV), 1e-20, 2, 1,
                                            "max", wg)),
    }[name]
    announce(f"opcheck {name}")
    torch.library.opcheck(op, args)


@pytest.mark.parametrize("name", ["experts", "layer", "router"])
def test_opcheck_of_rows_in_a_batch(decode, name):
    """x [B, S, D]: the rows come back flat, as the ops' shapes say."""
    importlib.import_module("torchtitan-ascend_amd.library")
    rng = np.random.default_rng(2)
    E, K, D, H = 4, 2, 96, 64
    w, _ = build(decode, rng, E, D, H, 16)
    x, wr, wg = weights(rng, 2, 3, D, scale=1.0), weights(rng, E, D), weights(rng, 1, D)
    idx = torch.from_numpy(np.argsort(rng.random((2, 3, E)), axis=2)[..., :K].copy()).to(DEV)
    ops = torch.ops.ttamd
    route = ("softmax", True, 1.0, None, 1e-20, None, None, "top2")
    op, args = {
        "experts": (ops.experts_decode, (x, torch.rand(2, 3, K, device=DEV), idx, *w, H, False, None)),
        "layer": (ops.moe_decode, (x, wr, *w, K, H, *route, False, None)),
        "router": (ops.router_decode, (x, wr, K, *route, wg)),
    }[name]
    announce(f"opcheck rows in a batch {name}")
    torch.library.opcheck(op, args)


# ---------------------------------------------------------------------------
# Prompts
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("T,E,K", [(65, 257, 2), (65, 300, 8), (200, 1024, 16), (130, 512, 1)])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("form", ["plain", "groups", "bias"])
def test_prompts_of_many_experts(decode, functional, T, E, K, bits, form):
    """The prompt's path takes as many experts as the few-token layer.  A logit is the
    bf16 of an fp32 sum, within b = 2^-8 |z| + (D + 8) 2^-24 sum |x w| (1 + 2^-8) of the
    64-bit z; picks are right within b, scores within a factor e^(2 b) and fp32."""
    rng = np.random.default_rng(T + E)
    D, H = 128, 128
    w, wb = build(decode, rng, E, D, H, bits)
    x, wr = weights(rng, T, D, scale=1.0), weights(rng, E, D)
    kw, func = {}, "softmax"
    if form == "groups":
        G = 4 if E % 4 == 0 else 1
        kw = dict(num_groups=G, topk_groups=max(1, G // 2), group_score="max")
    if form == "bias":
        kw, func = dict(expert_bias=torch.randn(E, device=DEV) * 0.05), "sigmoid"
    announce(f"prompt T={T} E={E} K={K} bits={bits} {form}")
    out, s, i = functional.moe_decode(x, wr, *w, K, func, **kw)
    with torch.no_grad():
        assert torch.equal(out, functional.moe_experts_forward(x, s, i, *wb, E, False))
    z = x.double() @ wr.double().t()
    size = x.double().abs() @ wr.double().abs().t()
    b = (2.0 ** -8 * z.abs() + (1 + 2.0 ** -8) * (D + 8) * 2.0 ** -24 * size).amax().item()
    p = torch.softmax(z, 1) if func == "softmax" else torch.sigmoid(z)
    near = np.exp(2 * b) * (1 + 2.0 ** -20)
    ratio = s.double() / p.gather(1, i)
    assert ratio.max() <= near and ratio.min() >= 1 / near
    # selection values: b moves a sigmoid by at most b / 4, a softmax score by the factor above
    v = p if form != "bias" else p + kw["expert_bias"].double()
    slack = b / 4 + 2.0 ** -20 if form == "bias" else (near - 1) * p.amax().item()
    if form == "groups" and kw["num_groups"] > 1:
        best = v.view(T, kw["num_groups"], -1).amax(2)
        kept = torch.zeros_like(best, dtype=torch.bool).scatter_(1, i // (E // kw["num_groups"]), True)
        assert (kept.sum(1) <= kw["topk_groups"]).all()
        last = best.topk(kw["topk_groups"], 1).values[:, -1]
        assert (torch.where(kept, best, torch.inf).amin(1) >= last - 2 * slack).all()
        v = torch.where(kept.repeat_interleave(E // kw["num_groups"], 1), v, -torch.inf)
    worst = v.gather(1, i).amin(1)
    rest = v.scatter(1, i, -torch.inf).amax(1)
    assert (rest - worst <= 2 * slack).all()
    assert (i.sort(1).values.diff(dim=1) > 0).all()  # no expert twice


@pytest.mark.parametrize("option", ["bf16", "e2m1"])
def test_module_of_many_choices(option):
    """More than 16 choices a token: the module's option changes nothing."""
    pkg = importlib.import_module("torchtitan-ascend_amd")
    E, K, D, H, T = 40, 20, 128, 64, 7
    rng = np.random.default_rng(3)
    idx = torch.from_numpy(np.argsort(rng.random((1, T, E)), axis=2)[..., :K].copy()).to(DEV)
    scores, x = torch.rand(1, T, K, device=DEV), weights(rng, 1, T, D, scale=1.0)
    w13, w2 = weights(rng, E, 2 * H, D), weights(rng, E, D, H)
    out = []
    for o in (None, option):
        m = pkg.HipGroupedExperts(pkg.HipGroupedExperts.Config(
            dim=D, hidden_dim=H, num_experts=E, decode_weights=o,
            token_dispatcher=pkg.HipTokenDispatcher.Config(num_experts=E, top_k=K))).to(DEV).bfloat16()
        with torch.no_grad():
            m.w13.copy_(w13)
            m.w2.copy_(w2)
            if o == "e2m1":
                m.pack_weights()
            announce(f"module K={K} {o}")
            out.append(m(x, scores, idx))
    assert torch.equal(*out)
