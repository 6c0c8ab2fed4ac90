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
from test_gpu_decode import BF16, build, check_product, layer_ref, weights

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


@pytest.mark.parametrize("T", [64, 65])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("Hs", [0, 192])
def test_prompt_of_one_expert(decode, functional, T, bits, Hs):
    """Weights [N, K] are one expert's; widths that are multiples of 64."""
    rng = np.random.default_rng(T)
    D, H = 256, 192
    w, wb = build(decode, rng, 1, D, H, 16, Hs)
    w = [t.reshape(t.shape[-2:]) for t in w]
    if bits == 4:
        w = [decode.pack_e2m1(t) for t in w]
        wb = [decode.unpack_e2m1(p).view(t.shape) for p, t in zip(w, wb)]
    x, wr = weights(rng, T, D, scale=1.0), weights(rng, 1, D)
    announce(f"one expert T={T} bits={bits} Hs={Hs}")
    kw = dict(shared_w13=w[2], shared_w2=w[3]) if Hs else {}
    out, s, i = functional.moe_decode(x, wr, *w[:2], 1, **kw)
    assert (s == 1).all() and (i == 0).all()
    if T > 64:
        with torch.no_grad():
            want = functional.moe_experts_forward(x, s, i, *wb[:2], 1, False)
            want = functional.shared_expert_combine(want, x, *wb[2:]) if Hs else want
        assert torch.equal(out, want)
        return
    ref, bound = layer_ref(x, s, i, *wb[:2], False, None, wb[2:] or None)
    assert ((out.double() - ref).abs() - bound).max() <= 0


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


# ---------------------------------------------------------------------------
# What a call writes
# ---------------------------------------------------------------------------
GUARD = 4096


class Guarded:
    """A tensor between two guards, all of one byte value; written() after a call: which
    rows changed, with the guards checked."""

    def __init__(self, shape, dtype, fill=0xA5):
        n = int(np.prod(shape)) * dtype.itemsize
        self.raw = torch.full((2 * GUARD + n,), fill, dtype=torch.uint8, device=DEV)
        self.fill, self.t = fill, self.raw[GUARD:GUARD + n].view(dtype).view(shape)

    def check(self, rows):
        """The guards and all rows but the given ones hold the fill, bit for bit."""
        torch.cuda.synchronize()
        assert (self.raw[:GUARD] == self.fill).all() and (self.raw[-GUARD:] == self.fill).all()
        left = torch.ones(self.t.shape[0], dtype=torch.bool)
        left[rows] = False
        assert (self.t.view(torch.uint8).cpu()[left] == self.fill).all()


def call(name, *args):
    lib = importlib.import_module("torchtitan-ascend_amd._lib")
    lib.call(name, *(a.data_ptr() if isinstance(a, torch.Tensor) else a for a in args),
             torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("counts,N,K", [
    ([1], 40, 64), ([0, 3, 0, 1], 97, 1056), ([5, 0, 17, 64, 65, 2], 131, 512), ([0, 0, 0], 32, 32),
    ([1] * 60, 1536, 2048),
    ([200, 1, 300], 31, 160), ([2] * 20, 18, 96), ([4, 3] * 8, 50, 288), ([30] * 5, 75, 544), ([100], 1003, 128)])
@pytest.mark.parametrize("past", [0, 1, 5, 70])
def test_rows_behind_the_last_run_stay(decode, counts, N, K, past):
    """Rows at or past offs[-1], and what lies in front of and behind the output, hold
    what they held."""
    rng = np.random.default_rng(sum(counts) + N)
    M, E = sum(counts) + past, len(counts)
    x, p = weights(rng, M, K, scale=1.0), decode.pack_e2m1(weights(rng, E, N, K))
    offs = torch.tensor(counts, device=DEV).cumsum(0).int()
    announce(f"rows behind counts={counts[:8]} N={N} K={K} past={past}")
    out = Guarded((M, N), BF16)
    call("ttamd_grouped_mm_e2m1", x, p.codes, p.exponents, offs, None, 0, M, E, N, K, out.t)
    out.check(slice(0, sum(counts)))
    w, r = decode.unpack_e2m1(p), 0
    for e, c in enumerate(counts):
        if c:
            check_product(x[r:r + c], w[e], out.t[r:r + c])
        r += c


def test_offsets_out_of_order_leave_rows(decode):
    """Ends that fall, pass the rows or are negative: rows of no run, and all around the
    output, stay."""
    rng = np.random.default_rng(0)
    E, M, N, K = 5, 12, 49, 96
    p, x = decode.pack_e2m1(weights(rng, E, N, K)), weights(rng, M, K, scale=1.0)
    w = decode.unpack_e2m1(p)
    for offs, runs in (([-3, 4, 2, 99, 99], {1: (0, 4), 3: (2, 12)}), ([0, 0, -5, -1, 3], {4: (0, 3)}),
                       ([7, 5, 5, 2, 2], {0: (0, 7)}), ([-9, -9, -9, -9, -9], {}),
                       ([2 ** 31 - 1, -2 ** 31, 1, 3, 3], {0: (0, 12), 2: (0, 1), 3: (1, 3)})):
        announce(f"offsets {offs}")
        out = Guarded((M, N), BF16)
        ends = torch.tensor(offs, dtype=torch.int32, device=DEV)
        call("ttamd_grouped_mm_e2m1", x, p.codes, p.exponents, ends, None, 0, M, E, N, K, out.t)
        rows = sorted({r for a, b in runs.values() for r in range(a, b)})
        out.check(rows)
        for e, (a, b) in runs.items():  # (rows of two runs hold either's)
            own = [r for r in range(a, b) if sum(lo <= r < hi for lo, hi in runs.values()) == 1]
            if own:
                check_product(x[own], w[e], out.t[own])


@pytest.mark.parametrize("M,N,K", [(1, 1, 32), (1, 5121, 160), (3, 17, 96), (13, 1001, 1440), (16, 33, 512),
                                   (17, 31, 288), (40, 65, 96), (64, 15, 1056), (100, 130, 128)])
def test_dense_products_write_their_rows_alone(decode, M, N, K):
    rng = np.random.default_rng(M + N)
    x, p, b = weights(rng, M, K, scale=1.0), decode.pack_e2m1(weights(rng, N, K)), Guarded((N,), BF16, 0x7F)
    b.t.copy_(weights(rng, N))
    announce(f"dense M={M} N={N} K={K}")
    out = Guarded((M, N), BF16)
    call("ttamd_grouped_mm_e2m1", x, p.codes, p.exponents, None, b.t, 0, M, 1, N, K, out.t)
    out.check(slice(0, M))
    check_product(x, decode.unpack_e2m1(p)[0], out.t, b.t)  # (the bias' guards are NaN)


@pytest.mark.parametrize("E,N,K", [(1, 1, 32), (3, 17, 160), (2, 15, 1056), (1, 33, 96), (2, 100, 544)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_packing_writes_its_tiles_alone(decode, E, N, K, dtype):
    rng = np.random.default_rng(N + K)
    w = weights(rng, E, N, K).to(dtype)
    want = decode.pack_e2m1(w)
    codes, exps = (Guarded(s, torch.uint8) for s in decode._shapes(E, N, K))
    out = Guarded((E, N, K), BF16)
    announce(f"pack E={E} N={N} K={K} {dtype}")
    call("ttamd_pack_e2m1", w, int(dtype == torch.float32), E, N, K, codes.t, exps.t)
    call("ttamd_unpack_e2m1", codes.t, exps.t, E, N, K, out.t)
    for g in (codes, exps, out):
        g.check(slice(0, E))
    assert torch.equal(codes.t, want.codes) and torch.equal(exps.t, want.exponents)
    assert torch.equal(out.t, decode.unpack_e2m1(want))


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("T,E,K,D,H,shared", [(1, 8, 2, 160, 96, 0), (5, 8, 2, 288, 32, 64), (33, 3, 3, 96, 64, 0),
                                              (64, 40, 16, 64, 32, 32), (64, 2, 1, 2080, 288, 96)])
def test_the_layer_writes_its_rows_and_its_workspace_alone(decode, T, E, K, D, H, shared, bits):
    lib = importlib.import_module("torchtitan-ascend_amd._lib").load()
    rng = np.random.default_rng(T + D)
    w, _ = build(decode, rng, E, D, H, bits, shared)
    x, wr = weights(rng, T, D, scale=1.0), weights(rng, E, D)
    tensors = [t for p in w for t in ((p.codes, p.exponents) if bits == 4 else (p, None))]
    tensors += [None] * (8 - len(tensors))
    announce(f"layer writes T={T} E={E} D={D} bits={bits}")
    out, scores, idx = Guarded((T, D), BF16), Guarded((T, K), torch.float32), Guarded((T, K), torch.int64)
    nbytes = lib.ttamd_moe_decode_workspace_bytes(T, D, H, E, K, shared)
    ws = Guarded((nbytes,), torch.uint8)
    call("ttamd_moe_decode", x, T, D, H, E, K, wr, None, 1, 1, 0, 0, 0, 1e-20, 1.0, 0, float("nan"), *tensors[:4],
         shared, *tensors[4:], None, scores.t, idx.t, out.t, ws.t, nbytes)
    for g in (out, scores, idx):
        g.check(slice(0, T))
    ws.check(slice(0, nbytes))
    want = decode.moe_decode(x, wr, *w[:2], K, shared_w13=w[2] if shared else None, shared_w2=w[3] if shared else None)
    equal((out.t, scores.t, idx.t), want)


# ---------------------------------------------------------------------------
# Every kernel that sizes choose
# ---------------------------------------------------------------------------
def gpu_weights(gen, *shape, scale=0.05):
    return (torch.randn(*shape, device=DEV, generator=gen) * scale).to(BF16)


# T, E, K, D, H, Hs; on 256 CUs these take each ring of both products in either type
FORMS16 = [
    (1, 4, 1, 96, 2080, 0), (1, 4, 1, 96, 288, 288), (1, 4, 3, 2080, 2080, 0), (1, 4, 1, 2080, 96, 288),
    (1, 4, 2, 2880, 1440, 0), (1, 2, 2, 4096, 2080, 0), (1, 4, 1, 4128, 2080, 0), (1, 4, 1, 4128, 96, 288),
    (1, 4, 1, 6400, 2080, 0), (1, 4, 1, 6400, 96, 288), (12, 4, 4, 2080, 1056, 64), (16, 4, 3, 96, 2080, 0),
    (16, 4, 3, 2080, 2080, 0), (17, 4, 1, 2080, 2080, 0), (17, 4, 1, 2080, 96, 288), (9, 1, 1, 4096, 1056, 0),
    (17, 4, 1, 4128, 2080, 0), (17, 4, 1, 4128, 96, 288), (17, 4, 1, 6400, 2080, 0), (9, 1, 1, 7168, 544, 0),
    (17, 4, 1, 6400, 96, 288), (24, 4, 2, 96, 544, 288), (24, 128, 12, 6400, 96, 0), (32, 128, 16, 5120, 64, 0),
    (32, 128, 16, 7168, 96, 0), (33, 4, 1, 96, 2080, 0), (33, 4, 1, 96, 288, 64), (33, 60, 13, 2080, 288, 0),
    (33, 128, 14, 4128, 96, 0), (33, 128, 15, 2080, 96, 64), (33, 256, 16, 2080, 96, 0), (48, 128, 9, 4128, 96, 288),
    (48, 128, 12, 96, 96, 64), (63, 16, 16, 96, 544, 64), (63, 60, 6, 2080, 288, 64), (63, 64, 4, 6400, 96, 64),
    (63, 128, 9, 96, 288, 0), (64, 16, 14, 2080, 544, 0), (64, 16, 16, 128, 96, 96), (64, 256, 9, 96, 96, 288),
    (64, 256, 10, 96, 288, 0),
]
FORMS4 = [
    (1, 4, 1, 96, 2080, 0), (1, 4, 1, 96, 288, 288), (1, 4, 3, 2080, 2080, 0), (1, 4, 1, 2080, 96, 288),
    (1, 4, 2, 2880, 1440, 0), (1, 2, 2, 4096, 2080, 0), (1, 4, 1, 4128, 2080, 0), (1, 4, 1, 4128, 96, 288),
    (9, 4, 1, 96, 2080, 0), (9, 4, 1, 96, 288, 288), (9, 4, 1, 2080, 2080, 0), (9, 4, 1, 2080, 96, 288),
    (5, 2, 1, 2880, 1056, 0), (5, 2, 1, 4096, 1056, 0), (16, 4, 1, 2880, 1056, 96), (9, 4, 1, 4128, 2080, 0),
    (9, 4, 1, 4128, 96, 288), (17, 4, 1, 96, 2080, 0), (17, 4, 1, 96, 288, 288), (63, 256, 9, 96, 288, 0),
    (63, 512, 14, 96, 96, 0), (4, 60, 4, 2080, 1056, 32), (8, 60, 2, 4128, 544, 0), (16, 64, 4, 2880, 1440, 0),
]


@pytest.mark.parametrize("bits,form", [(16, f) for f in FORMS16] + [(4, f) for f in FORMS4])
@pytest.mark.parametrize("before", [False, True])
def test_every_stream(decode, bits, form, before):
    T, E, K, D, H, Hs = form
    gen = torch.Generator(DEV).manual_seed(T + D + H)
    w = [gpu_weights(gen, E, 2 * H, D), gpu_weights(gen, E, D, H)]
    w += [gpu_weights(gen, 2 * Hs, D), gpu_weights(gen, D, Hs)] if Hs else []
    wb, limit = w, 0.9 if before else None
    if bits == 4:
        w = [decode.pack_e2m1(t) for t in w]
        wb = [decode.unpack_e2m1(p).view(t.shape) for p, t in zip(w, wb)]
    x = gpu_weights(gen, T, D, scale=1.0)
    idx = torch.rand(T, E, device=DEV, generator=gen).argsort(1)[:, :K].contiguous()
    scores = torch.rand(T, K, device=DEV, generator=gen)
    announce(f"streams T={T} E={E} K={K} D={D} H={H} Hs={Hs} bits={bits} before={before}")
    y = decode.experts_decode(x, scores, idx, *w[:2], before, limit, *(w[2:] or (None, None)))
    ref, bound = layer_ref(x, scores, idx, *wb[:2], before, limit, wb[2:] or None)
    off = ((y.double() - ref).abs() - bound).max().item()
    assert off <= 0, f"{off:.3e} past the bound"
    again = decode.experts_decode(x, scores, idx, *w[:2], before, limit, *(w[2:] or (None, None)))
    assert torch.equal(y, again)


@pytest.mark.parametrize("T,E,K,groups", [
    (61, 8, 1, None), (9, 64, 12, None), (32, 128, 8, None), (32, 128, 12, (4, 2)), (20, 160, 6, (8, 3)),
    (20, 192, 16, None),
    (17, 256, 8, (8, 4)), (17, 256, 16, None), (9, 200, 8, (8, 4)), (9, 256, 16, (64, 20)), (5, 300, 4, (3, 2)),
    (5, 512, 16, None), (33, 1024, 8, (64, 7)), (33, 1024, 16, None), (7, 990, 8, (33, 4)), (64, 1023, 16, (33, 20)),
    (2, 961, 3, (31, 1)), (64, 63, 3, (63, 5)),
])
@pytest.mark.parametrize("func", ["softmax", "sigmoid"])
def test_every_plan(decode, T, E, K, groups, func):
    """The selection within the plan against the router's own kernel, and the stage on
    the plan's picks against the one that is given them."""
    rng = np.random.default_rng(T + E)
    D, H = 64, 32
    w, _ = build(decode, rng, E, D, H, 16)
    x, wr = weights(rng, T, D, scale=1.0), weights(rng, E, D)
    kw = {} if groups is None else dict(num_groups=groups[0], topk_groups=groups[1])
    bias = torch.randn(E, device=DEV) * 0.05 if T % 2 else None
    announce(f"plan T={T} E={E} K={K} {groups} {func}")
    out, s, i = decode.moe_decode(x, wr, *w, K, func, True, 2.5, bias, **kw)
    equal((s, i), decode.router_decode(x, wr, K, func, True, 2.5, bias, **kw)[:2])
    assert torch.equal(out, decode.experts_decode(x, s, i, *w))
