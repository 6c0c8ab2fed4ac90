"""The operators around the expert stage used together: the MoE block (norm,
group-limited router, experts, combine with norm, gate, residual and the next
norm), in training with and without 8-bit activation checkpoints, in
inference, captured as a graph, and through the converted module; against a
64-bit restatement with the GPU's own picks, within the path's 2e-2 for whole
layers (bf16 intermediates), per row and per expert."""
from __future__ import annotations

import importlib

import numpy as np
import pytest
import torch

from gpu_util import DEV, announce, assert_close, bf16_dev, rand_bf16, to_np

BF16 = torch.bfloat16
EPS = 1e-6
TOL = 2e-2


def F():
    return importlib.import_module("torchtitan-ascend_amd.functional")


def inputs(rng, T, D, H, E, gate="token", x_dtype=BF16):
    f32 = lambda *s, m=0.0, sd=1.0: torch.from_numpy((rng.standard_normal(s) * sd + m).astype(np.float32)).to(DEV)  # noqa: E731
    shape = {"none": None, "token": (T, 1), "channel": (1, D)}[gate]
    return dict(x=f32(T, D, sd=2.0).to(x_dtype), w_router=bf16_dev(rand_bf16(rng, (E, D), 0.05)),
                w13=bf16_dev(rand_bf16(rng, (E, 2 * H, D), 0.05)), w2=bf16_dev(rand_bf16(rng, (E, D, H), 0.05)),
                pre_weight=f32(D, m=1.0, sd=0.2), post_weight=f32(D, m=1.0, sd=0.2),
                next_weight=f32(D, m=1.0, sd=0.2), gate=None if shape is None else f32(*shape),
                expert_bias=f32(E, sd=0.02))


def call(c, K, **o):
    c = dict(c)
    x, wr, w13, w2 = (c.pop(k) for k in ("x", "w_router", "w13", "w2"))
    return F().moe_block(x, wr, w13, w2, K, gate_func="sigmoid", residual_scale=0.5, eps=EPS, **c, **o)


def rms(v, w):
    return v / torch.sqrt(v.square().mean(1, keepdim=True) + EPS) * w


def define(c, idx, func, norm, scale, before, limit):
    """The block in 64 bits from leaves c, on given picks, and its router
    logits.  The gate Linear's output is bf16 by the router's contract,
    straight through for gradients."""
    st = lambda v: v + (v.detach().to(BF16).double() - v.detach())  # noqa: E731
    x = c["x"]
    h = st(rms(x, c["pre_weight"]))
    z = st(h @ c["w_router"].t())
    z.retain_grad()
    p = torch.softmax(z, 1) if func == "softmax" else torch.sigmoid(z)
    s = p.gather(1, idx)
    if norm:
        s = s / (s.sum(1, keepdim=True) + 1e-20)
    s = s * scale
    H = c["w2"].shape[2]
    f = torch.zeros_like(x)
    for k in range(idx.shape[1]):
        for e in range(c["w13"].shape[0]):
            t = (idx[:, k] == e).nonzero(as_tuple=True)[0]
            if not len(t):
                continue
            r = h[t] * (s[t, k:k + 1] if before else 1.0)
            g = st(r) @ c["w13"][e].t()
            gate, up = st(g)[:, :H], st(g)[:, H:]
            if limit is not None:
                gate, up = gate.clamp(max=limit), up.clamp(-limit, limit)
            y = st(torch.nn.functional.silu(gate) * up) @ c["w2"][e].t()
            f = f.index_add(0, t, y * (1.0 if before else s[t, k:k + 1]))
    b = rms(st(f), c["post_weight"])
    if c["gate"] is not None:
        b = b * torch.sigmoid(c["gate"])
    u = x + 0.5 * b
    return u, rms(u, c["next_weight"]), z, h


CASES = [
    # T, D, H, E, K, groups, kept, func, norm, before, limit, gate
    (1, 128, 128, 8, 2, 4, 2, "sigmoid", True, False, None, "token"),
    (130, 256, 128, 16, 4, 4, 2, "sigmoid", True, False, None, "token"),
    (257, 256, 128, 12, 3, 3, 2, "softmax", False, False, 0.5, "channel"),
    (200, 128, 256, 8, 1, 4, 3, "sigmoid", False, True, None, "none"),
]


def routing(ops, c, K, func, norm, groups):
    """The block's own picks (its router runs on bf16 h)."""
    h = ops.rms_norm(c["x"], c["pre_weight"], EPS)
    return ops.router_fused(h, c["w_router"], K, func, norm, 2.5, c["expert_bias"], **groups)[1]


@pytest.mark.gpu
@pytest.mark.parametrize("T,D,H,E,K,G,kept,func,norm,before,limit,gate", CASES)
@pytest.mark.parametrize("x_dtype", [BF16, torch.float32])
def test_block_forward_and_gradients(ops, T, D, H, E, K, G, kept, func, norm, before, limit, gate, x_dtype):
    rng = np.random.default_rng(T + D + E)
    c = inputs(rng, T, D, H, E, gate, x_dtype)
    groups = dict(num_groups=G, topk_groups=kept)
    kw = dict(score_func=func, route_norm=norm, route_scale=2.5, score_before_experts=before, swiglu_limit=limit,
              **groups)
    announce(f"moe_block T={T} D={D} E={E} K={K} {func} before={before} {x_dtype}")
    idx = routing(ops, c, K, func, norm, groups)
    names = [k for k in c if c[k] is not None and k != "expert_bias"]
    leaves = {k: c[k].clone().requires_grad_(True) for k in names}
    u, n = call({**c, **leaves}, K, **kw)
    du = torch.from_numpy(rng.standard_normal((T, D)).astype(np.float32)).to(DEV).to(x_dtype)
    dn = bf16_dev(rand_bf16(rng, (T, D)))
    torch.autograd.backward([u, n], [du, dn])
    # vectors (weights, gate) enter the reference expanded to [T, D]: the leaf's
    # gradient is then the terms that the vector's gradient sums
    vectors = [k for k in names if c[k].dim() == 1 or 1 in c[k].shape and k == "gate"]
    wide = {k: (None if c[k] is None else c[k].double()) for k in c}
    for k in vectors:
        wide[k] = wide[k].expand(T, D).clone()
    for k in names:
        wide[k].requires_grad_(True)
    ru, rn, z, h = define(wide, idx, func, norm, 2.5, before, limit)
    torch.autograd.backward([ru, rn], [du.double(), dn.double()])
    ref = {k: wide[k].grad for k in names}
    assert u.dtype == x_dtype and n.dtype == BF16
    assert_close(to_np(u), ru.detach().float().cpu().numpy(), TOL, "u")
    assert_close(to_np(n), rn.detach().float().cpu().numpy(), TOL, "n")
    cpu = lambda t: t.detach().float().cpu().numpy()  # noqa: E731
    for k in names:
        got = to_np(leaves[k].grad)
        if k in vectors or k == "w_router":
            # sums of products whose terms cancel.  Every factor is within the
            # path's 2e-2 of its row's largest entry (not of itself), so a sum
            # is within 2e-2 of the largest sum of |terms|
            if k == "w_router":
                want, size = ref[k], z.grad.abs().t() @ h.abs()
            else:
                axis = 1 if c[k].shape == (T, 1) else 0
                want, size = ref[k].sum(axis), ref[k].abs().sum(axis)
            err = np.abs(got.reshape(-1) - cpu(want).reshape(-1)).max() / cpu(size).max()
            assert err < TOL, f"d{k}: {err:.3e}"
        else:
            assert_close(got, cpu(ref[k]), TOL, f"d{k}")
    # inference: the same block, the norms inside the combine
    with torch.no_grad():
        ui, ni = call(c, K, **kw)
        assert ui.dtype == x_dtype
        assert_close(to_np(ui), ru.detach().float().cpu().numpy(), TOL, "inference u")
        assert_close(to_np(ni), rn.detach().float().cpu().numpy(), TOL, "inference n")


@pytest.mark.gpu
@pytest.mark.parametrize("T,D,H,E,K,before,limit,wdtype", [
    (150, 256, 128, 8, 4, False, None, torch.float32), (64, 128, 256, 4, 1, True, None, BF16),
    (300, 384, 128, 16, 2, False, 0.5, BF16), (1, 128, 128, 8, 8, False, None, torch.float32),
])
def test_checkpointed_experts(ops, T, D, H, E, K, before, limit, wdtype):
    """With 8-bit checkpoints the output is the plain path's and the gradients
    are those of the formulas at the stored activations: x, h and y restored
    from their codes, everything else 64 bits, within the path's 2e-2."""
    rng = np.random.default_rng(T + D + K)
    x = bf16_dev(rand_bf16(rng, (T, D)))
    w13 = bf16_dev(rand_bf16(rng, (E, 2 * H, D), 0.05)).to(wdtype)
    w2 = bf16_dev(rand_bf16(rng, (E, D, H), 0.05)).to(wdtype)
    idx = torch.from_numpy(np.argsort(rng.random((T, E)), axis=1)[:, :K].astype(np.int64)).to(DEV)
    sc = torch.from_numpy((rng.random((T, K)) * 0.8 + 0.2).astype(np.float32)).to(DEV)
    dout = bf16_dev(rand_bf16(rng, (T, D)))
    announce(f"checkpointed experts T={T} D={D} H={H} E={E} K={K} before={before} limit={limit} {wdtype}")

    def step(checkpoint):
        leaves = [t.clone().requires_grad_(True) for t in (x, sc, w13, w2)]
        out = F().moe_experts_forward(leaves[0], leaves[1], idx, leaves[2], leaves[3], E, before, limit,
                                      checkpoint=checkpoint)
        out.backward(dout)
        return out.detach(), [t.grad for t in leaves]

    plain, _ = step(None)
    out, (dx, dsc, dw13, dw2) = step("e4m3")
    torch.cuda.synchronize()
    assert_close(to_np(out), to_np(plain), 2.0 ** -7, "output")
    assert dw13.dtype == wdtype and dw2.dtype == wdtype
    # the stored values
    r = ops.route(idx, E, sc)
    restore = lambda t: ops.unpack_e4m3(ops.pack_e4m3(t))  # noqa: E731
    routed = ops.permute_rows(x, r, K, sc.reshape(-1) if before else None)
    a, h = ops.grouped_mm_swiglu(routed, w13.to(BF16), r.offs, limit, save_h=True)
    y = restore(ops.grouped_mm_unpermute(a, w2.to(BF16), r.offs)).double()
    hs = restore(h).double().requires_grad_(True)
    slot = r.sorted_indices.long()
    tok = slot // K
    s = sc.reshape(-1)[slot].double().unsqueeze(1)
    xs = restore(x).double()[tok]
    if before:
        xs = (xs.float() * s.float()).to(BF16).double()
    gate, up = hs[:, :H], hs[:, H:]
    if limit is not None:
        gate, up = gate.clamp(max=limit), up.clamp(-limit, limit)
    act = torch.nn.functional.silu(gate) * up
    go = dout.double()[tok]
    dy = go if before else go * s
    ex = torch.repeat_interleave(torch.arange(E, device=DEV), r.counts.long())
    w2d, w13d = w2.to(BF16).double(), w13.to(BF16).double()
    da = torch.stack([dy[i] @ w2d[ex[i]] for i in range(T * K)])
    (dh,) = torch.autograd.grad(act, hs, da)
    act = act.detach()
    rw2 = torch.zeros_like(w2d)
    rw13 = torch.zeros_like(w13d)
    for e in range(E):
        m = ex == e
        rw2[e] = dy[m].t() @ act[m]
        rw13[e] = dh[m].t() @ xs[m]
    dr = torch.stack([dh[i] @ w13d[ex[i]] for i in range(T * K)])
    rdx = torch.zeros(T, D, dtype=torch.float64, device=DEV).index_add(0, tok, dr * (s if before else 1.0))
    dots = (dr * restore(x).double()[tok] if before else go * y)
    rds = torch.zeros(T * K, dtype=torch.float64, device=DEV)
    rds[slot] = dots.sum(1)
    size = torch.zeros(T * K, dtype=torch.float64, device=DEV)
    size[slot] = dots.abs().sum(1)
    cpu = lambda t: t.float().cpu().numpy()  # noqa: E731
    assert_close(to_np(dw2), cpu(rw2), TOL, "dw2")
    assert_close(to_np(dw13), cpu(rw13), TOL, "dw13")
    assert_close(to_np(dx), cpu(rdx), TOL, "dx")
    err = (dsc.reshape(-1).double() - rds).abs() / size
    assert float(err.max()) < TOL


@pytest.mark.gpu
def test_checkpoint_memory_and_module(pkg):
    """The converted module with activation_checkpoint="e4m3": the same output,
    gradients for every input, and less than 0.45 of the bytes kept between
    forward and backward (x, routed, h, a, y in bf16 against x, h, y at 1 +
    1/128 byte: (2 D + 2 K (2 D + 3 H)) against 1.01 (D + K (2 H + D)), 0.31
    here, and a few index maps)."""
    P = importlib.import_module("torchtitan-ascend_amd.protocol")
    T, D, H, E, K = 4096, 512, 256, 16, 8
    kept, outs = [], []
    g = torch.Generator(device=DEV).manual_seed(3)
    x0 = torch.randn(1, T, D, device=DEV, generator=g).to(BF16)
    idx = torch.rand(T, E, device=DEV, generator=g).argsort(1)[:, :K]
    sc = torch.rand(T, K, device=DEV, generator=g)
    for mode in (None, "e4m3"):
        mc = P.ModelConfig()
        mc.moe = P.GroupedExperts.Config(
            dim=D, hidden_dim=H, num_experts=E,
            token_dispatcher=P.AllToAllTokenDispatcher.Config(num_experts=E, top_k=K, score_before_experts=False))
        pkg.HipGroupedExpertsConverter(pkg.HipGroupedExpertsConverter.Config(activation_checkpoint=mode)).convert(mc)
        pkg.HipTokenDispatcherConverter(pkg.HipTokenDispatcherConverter.Config()).convert(mc)
        assert mc.moe.activation_checkpoint == mode
        m = mc.moe.build().to(DEV).to(BF16)
        with torch.no_grad():
            gen = torch.Generator(device=DEV).manual_seed(4)
            m.w13.normal_(0, 0.05, generator=gen)
            m.w2.normal_(0, 0.05, generator=gen)
        x, s = x0.clone().requires_grad_(True), sc.clone().requires_grad_(True)
        announce(f"module with activation_checkpoint={mode}")
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        out = m(x, s, idx)
        torch.cuda.synchronize()
        kept.append(torch.cuda.memory_allocated() - before)
        outs.append(out.detach().clone())
        out.float().square().sum().backward()
        for t in (x, s, m.w13, m.w2):
            assert t.grad is not None and bool(t.grad.isfinite().all()) and bool(t.grad.any())
        del out, m, x, s
    assert_close(to_np(outs[1]), to_np(outs[0]), 2.0 ** -7, "output")
    assert kept[1] < 0.45 * kept[0], kept


@pytest.mark.gpu
@pytest.mark.parametrize("T,D,H,E,K,G,kept", [(64, 256, 128, 16, 4, 4, 2), (1, 128, 128, 8, 2, 4, 2),
                                              (2100, 512, 256, 32, 8, 8, 4)])
def test_block_graph_replays_equal_eager(ops, T, D, H, E, K, G, kept):
    """MoELayerGraph with the block around the layer: every replay equals the
    eager block on the same input, with eager work between the replays; two
    graphs in turn, each with buffers of its own."""
    MoELayerGraph = importlib.import_module("torchtitan-ascend_amd.graph").MoELayerGraph
    rng = np.random.default_rng(T + E)
    c = inputs(rng, T, D, H, E, "token")
    args = dict(score_func="sigmoid", route_norm=True, route_scale=2.5, num_groups=G, topk_groups=kept)
    block = {k: c[k] for k in ("pre_weight", "post_weight", "next_weight", "gate", "expert_bias")}
    announce(f"block graph T={T} D={D} E={E} K={K}")
    make = lambda: MoELayerGraph(c["x"], c["w_router"], c["w13"], c["w2"], K, gate_func="sigmoid",  # noqa: E731
                                 residual_scale=0.5, eps=EPS, **args, **block)
    graphs = [make(), make()]
    with torch.no_grad():
        for i in range(4):
            xs = [torch.from_numpy(rng.standard_normal((T, D)).astype(np.float32)).to(DEV).to(BF16) for _ in range(2)]
            outs = [g(x) for g, x in zip(graphs, xs)]
            for (u, n), x in zip(outs, xs):
                eu, en = call({**c, "x": x}, K, **args)
                torch.cuda.synchronize()
                assert torch.equal(u, eu) and torch.equal(n, en), f"replay {i}"
    # groups alone, without a block
    layer = MoELayerGraph(c["x"], c["w_router"], c["w13"], c["w2"], K, expert_bias=c["expert_bias"], **args)
    x = c["x"] * 0.5
    got = layer(x).clone()
    _, _, r = ops.router_route(x, c["w_router"], K, "sigmoid", True, 2.5, c["expert_bias"], num_groups=G,
                               topk_groups=kept)
    assert torch.equal(got, ops.experts_forward(x, r, c["w13"], c["w2"], K, False))


@pytest.mark.gpu
@pytest.mark.parametrize("T,D,K,before", [(1, 128, 1, False), (70, 256, 4, False), (90, 128, 3, True)])
def test_experts_rows_sum_to_the_layer(ops, T, D, K, before):
    """experts_forward(sum_rows=False): the same rows that the K-way sum adds,
    so their fp32 sum rounds to its output."""
    rng = np.random.default_rng(T + D)
    H, E = 128, 8
    x, wr = bf16_dev(rand_bf16(rng, (T, D))), bf16_dev(rand_bf16(rng, (E, D), 0.05))
    w13, w2 = bf16_dev(rand_bf16(rng, (E, 2 * H, D), 0.05)), bf16_dev(rand_bf16(rng, (E, D, H), 0.05))
    announce(f"experts rows T={T} D={D} K={K} before={before}")
    _, _, r = ops.router_route(x, wr, K, "sigmoid", False)
    out = ops.experts_forward(x, r, w13, w2, K, before)
    _, _, r = ops.router_route(x, wr, K, "sigmoid", False)
    rows = ops.experts_forward(x, r, w13, w2, K, before, sum_rows=False)
    assert rows.shape == (T * K, D)
    total = rows.view(T, K, D)[:, 0].float()
    for k in range(1, K):
        total = total + rows.view(T, K, D)[:, k].float()
    assert torch.equal(total.to(BF16), out)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["router_grouped", "router_topk", "router_topk_backward", "residual_norm",
                                  "residual_norm_plain", "rms_norm", "residual_norm_backward", "experts_packed",
                                  "experts_packed_before", "moe_block_forward"])
def test_opcheck(ops, name):
    importlib.import_module("torchtitan-ascend_amd.library")
    T_ = torch.ops.ttamd
    rng = np.random.default_rng(2)
    T, D, H, E, K = 40, 128, 128, 8, 2
    c = inputs(rng, T, D, H, E)
    rq = lambda t: t.detach().clone().requires_grad_(True)  # noqa: E731
    z = torch.randn(T, E, device=DEV)
    s, idx = ops.router_topk(z, K, "sigmoid", True, num_groups=4, topk_groups=2)
    r = ops.route(idx, E, s)
    _, _, st = ops.residual_norm(c["x"], c["x"], c["post_weight"], c["gate"], pre_weight=c["next_weight"],
                                 save_stats=True)
    flat = s.reshape(-1).contiguous()
    packed = lambda before: (rq(c["x"]), rq(flat), r.sorted_indices, r.inverse, r.sorted_scores,  # noqa: E731
                             r.offs.contiguous(), rq(c["w13"]), rq(c["w2"]), K, before, None, not before)
    op, args = {
        "router_grouped": (T_.router, (rq(c["x"]), rq(c["w_router"]), K, "sigmoid", True, 1.0, None, 1e-20, 4, 2,
                                       "max")),
        "router_topk": (T_.router_topk, (rq(z), K, "softmax", True, 1.0, None, 1e-20, 4, 2, "top2")),
        "router_topk_backward": (T_.router_topk_backward, (s, idx, z, "sigmoid", True, 1.0, 1e-20)),
        "residual_norm": (T_.residual_norm, (rq(c["x"]), rq(c["x"]), rq(c["post_weight"]), rq(c["gate"]), "sigmoid",
                                             0.5, rq(c["next_weight"]), EPS, True)),
        "residual_norm_plain": (T_.residual_norm, (c["x"], None, None, None, "identity", 1.0, None, EPS, False)),
        "rms_norm": (T_.rms_norm, (rq(c["x"]), rq(c["pre_weight"]), EPS, True)),
        "residual_norm_backward": (T_.residual_norm_backward, (c["x"], c["x"], c["x"], st, c["x"], c["post_weight"],
                                                               c["gate"], "identity", 1.0, c["next_weight"])),
        "experts_packed": (T_.experts_packed, packed(False)),
        "experts_packed_before": (T_.experts_packed, packed(True)),
        "moe_block_forward": (T_.moe_block_forward, (
            c["x"], c["w_router"], c["w13"], c["w2"], K, c["pre_weight"], c["post_weight"], c["gate"], "sigmoid", 0.5,
            c["next_weight"], EPS, "sigmoid", True, 1.0, None, 4, 2, "top2", False, None)),
    }[name]
    announce(f"opcheck ttamd::{name}")
    torch.library.opcheck(op, args)


@pytest.mark.gpu
def test_calls_on_two_streams(ops):
    """The same operators on two streams at once, with nothing between them:
    each gives what it gives alone."""
    rng = np.random.default_rng(31)
    c = [inputs(rng, 700, 512, 256, 16) for _ in range(2)]
    kw = dict(score_func="sigmoid", route_norm=True, num_groups=4, topk_groups=2)
    idx = [routing_idx(ops, v, 4, kw) for v in c]
    sc = torch.rand(700, 4, device=DEV)

    def work(v, i):
        with torch.no_grad():
            u, n = call(v, 4, **kw)
        leaves = [v["x"].clone().requires_grad_(True), v["w13"].clone().requires_grad_(True)]
        out = F().moe_experts_forward(leaves[0], sc, i, leaves[1], v["w2"], 16, False, checkpoint="e4m3")
        out.backward(u)
        return u, n, out.detach(), leaves[0].grad, leaves[1].grad

    announce("two streams")
    alone = [work(v, i) for v, i in zip(c, idx)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in c]
    for _ in range(3):
        both = []
        for s, v, i in zip(streams, c, idx):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                both.append(work(v, i))
        torch.cuda.synchronize()
        for a, b in zip(alone, both):
            for x, y in zip(a, b):
                assert torch.equal(x, y)


def routing_idx(ops, c, K, kw):
    h = ops.rms_norm(c["x"], c["pre_weight"], EPS)
    return ops.router_fused(h, c["w_router"], K, kw["score_func"], kw["route_norm"],
                            num_groups=kw["num_groups"], topk_groups=kw["topk_groups"])[1]


@pytest.mark.gpu
def test_repeatable(ops):
    """The same call gives the same bits: no sum depends on an arrival order."""
    rng = np.random.default_rng(32)
    c = inputs(rng, 3000, 512, 256, 16, "channel")
    kw = dict(score_func="softmax", num_groups=4, topk_groups=3, checkpoint="e4m3")

    def step():
        names = [k for k in c if k != "expert_bias"]
        leaves = {k: c[k].clone().requires_grad_(True) for k in names}
        u, n = call({**c, **leaves}, 4, **kw)
        torch.autograd.backward([u, n], [c["x"], c["x"]])
        return [u, n] + [leaves[k].grad for k in names]

    announce("repeatable")
    first = step()
    for _ in range(3):
        for a, b in zip(first, step()):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_block_without_tokens(ops):
    rng = np.random.default_rng(33)
    c = inputs(rng, 4, 128, 128, 8)
    c["x"], c["gate"] = c["x"][:0], c["gate"][:0]
    announce("block without tokens")
    with torch.no_grad():
        u, n = call(c, 2, score_func="sigmoid", num_groups=4, topk_groups=2)
    assert u.shape == (0, 128) and n.shape == (0, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_block_gradients_without_tokens(ops, checkpoint):
    """No tokens: empty outputs and exact zeros for every weight."""
    rng = np.random.default_rng(34)
    c = inputs(rng, 4, 128, 128, 8, "channel")
    c["x"] = c["x"][:0]
    names = [k for k in c if k != "expert_bias"]
    leaves = {k: c[k].clone().requires_grad_(True) for k in names}
    announce(f"block gradients without tokens, checkpoint {checkpoint}")
    u, n = call({**c, **leaves}, 2, score_func="sigmoid", num_groups=4, topk_groups=2, checkpoint=checkpoint)
    (u.float().sum() + n.float().sum()).backward()
    for k in names:
        g = leaves[k].grad
        assert g is not None and g.shape == c[k].shape and not g.any(), k


@pytest.mark.gpu
@pytest.mark.parametrize("before", [False, True])
def test_gradients_of_some_inputs_are_those_of_all(ops, before):
    """Whatever is asked for beside it, an input's gradient has the same bits;
    the upstream gradient is a broadcast one."""
    rng = np.random.default_rng(35)
    c = inputs(rng, 300, 256, 128, 8)
    sc = torch.rand(300, 4, device=DEV)
    idx = torch.rand(300, 8, device=DEV).argsort(1)[:, :4]
    names = ("x", "scores", "w13", "w2")

    def grads(wanted):
        t = dict(x=c["x"].clone(), scores=sc.clone(), w13=c["w13"].clone(), w2=c["w2"].clone())
        for k in wanted:
            t[k].requires_grad_(True)
        F().moe_experts_forward(t["x"], t["scores"], idx, t["w13"], t["w2"], 8, before,
                                checkpoint="e4m3").sum().backward()
        return {k: t[k].grad for k in wanted}

    announce("gradients of some inputs")
    every = grads(names)
    for k in names:
        assert torch.equal(grads((k,))[k], every[k]), k


def test_module_refuses_an_unknown_checkpoint(pkg):
    P = importlib.import_module("torchtitan-ascend_amd.protocol")
    mc = P.ModelConfig()
    mc.moe = P.GroupedExperts.Config(
        dim=128, hidden_dim=128, num_experts=4,
        token_dispatcher=P.AllToAllTokenDispatcher.Config(num_experts=4, top_k=1, score_before_experts=False))
    pkg.HipGroupedExpertsConverter(pkg.HipGroupedExpertsConverter.Config(activation_checkpoint="int8")).convert(mc)
    with pytest.raises(ValueError, match="activation_checkpoint"):
        mc.moe.build()


def test_module_refuses_a_checkpoint_with_another_dispatcher(pkg):
    P = importlib.import_module("torchtitan-ascend_amd.protocol")
    mc = P.ModelConfig()
    mc.moe = P.GroupedExperts.Config(
        dim=128, hidden_dim=128, num_experts=4,
        token_dispatcher=P.AllToAllTokenDispatcher.Config(num_experts=4, top_k=1, score_before_experts=False))
    pkg.HipGroupedExpertsConverter(pkg.HipGroupedExpertsConverter.Config(activation_checkpoint="e4m3")).convert(mc)
    m = mc.moe.build()
    with pytest.raises(NotImplementedError, match="HipTokenDispatcher"):
        m(torch.zeros(1, 2, 128), torch.zeros(1, 2, 1), torch.zeros(1, 2, 1, dtype=torch.int64))


def test_unknown_checkpoint_refused_without_autograd():
    with torch.no_grad(), pytest.raises(ValueError, match="checkpoint"):
        F().moe_experts_forward(torch.zeros(2, 128), torch.zeros(2, 1), torch.zeros(2, 1, dtype=torch.int64),
                                torch.zeros(4, 256, 128), torch.zeros(4, 128, 128), 4, False, checkpoint="int8")


def test_experts_rows_refusals():
    import ctypes

    L = importlib.import_module("torchtitan-ascend_amd._lib").load()
    p, nan = ctypes.c_void_p(256), float("nan")
    need = L.ttamd_moe_experts_rows_workspace_bytes(64, 128, 128, 4, 2, 0)
    assert need <= L.ttamd_moe_experts_forward_workspace_bytes(64, 128, 128, 4, 2, 0)
    args = lambda D, ws: (p, 64, D, 128, 4, 2, p, p, p, 0, nan, p, p, p, None, 0, p, ws, None)  # noqa: E731
    assert L.ttamd_moe_experts_rows(*args(192, need)) == 1
    assert "ttamd_moe_experts_rows: dim" in L.ttamd_last_error().decode()
    assert L.ttamd_moe_experts_rows(*args(128, need - 1)) == 1
    assert "workspace" in L.ttamd_last_error().decode()


def _experts(E, D=128, H=128, device="cpu"):
    bf = lambda *n: torch.zeros(*n, dtype=BF16, device=device)  # noqa: E731
    return bf(E, 2 * H, D), bf(E, D, H)


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("E", [4, 16])
def test_block_refuses_a_gate_of_other_experts(grad, E):
    """A router of 8 experts before 4 or 16: the offsets and the tile table that
    it makes are not those the expert stage reads."""
    w13, w2 = _experts(E)
    x = torch.zeros(2, 128, dtype=BF16, requires_grad=grad)
    with torch.set_grad_enabled(grad), pytest.raises(ValueError, match="experts"):
        F().moe_block(x, torch.zeros(8, 128, dtype=BF16), w13, w2, 2)


@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
@pytest.mark.parametrize("grad", [False, True])
def test_expert_stage_refuses_another_number_of_experts(grad, checkpoint):
    w13, w2 = _experts(4)
    x = torch.zeros(2, 128, dtype=BF16, requires_grad=grad)
    with torch.set_grad_enabled(grad), pytest.raises(ValueError, match="experts"):
        F().moe_experts_forward(x, torch.zeros(2, 1), torch.zeros(2, 1, dtype=torch.int64), w13, w2, 8, False,
                                checkpoint=checkpoint)


@pytest.mark.gpu
@pytest.mark.parametrize("sum_rows", [True, False])
def test_experts_forward_refuses_a_routing_of_other_experts(ops, sum_rows):
    """Refused on the host, with a tile plan and without."""
    x = torch.zeros(6, 128, dtype=BF16, device=DEV)
    idx = torch.arange(6, device=DEV).view(6, 1)
    w13, w2 = _experts(8, device=DEV)
    for E in (4, 16):
        announce(f"experts_forward on a routing of {E} experts")
        for r in (ops.route(idx % E, E, torch.ones(6, 1, device=DEV)),
                  ops.router_route(x, torch.zeros(E, 128, dtype=BF16, device=DEV), 1)[2]):
            with pytest.raises(ValueError, match="experts"):
                ops.experts_forward(x, r, w13, w2, 1, False, sum_rows=sum_rows)


@pytest.mark.parametrize("grad", [False, True])
def test_block_refuses_an_unknown_checkpoint(grad):
    """With autograd and without, where nothing is kept."""
    w13, w2 = _experts(4)
    x = torch.zeros(2, 128, dtype=BF16, requires_grad=grad)
    with torch.set_grad_enabled(grad), pytest.raises(ValueError, match="checkpoint"):
        F().moe_block(x, torch.zeros(4, 128, dtype=BF16), w13, w2, 2, checkpoint="int8")


@pytest.mark.gpu
@pytest.mark.parametrize("block", [True, False])
def test_graph_of_an_fp32_stream(block):
    """What moe_block takes, the graph of it takes: an fp32 residual stream,
    with norms and without; every replay equals the eager block."""
    MoELayerGraph = importlib.import_module("torchtitan-ascend_amd.graph").MoELayerGraph
    rng = np.random.default_rng(36)
    T, D, K = 70, 256, 4
    c = inputs(rng, T, D, 128, 8, "channel", torch.float32)
    names = ("pre_weight", "post_weight", "next_weight", "gate") if block else ()
    how = dict(gate_func="sigmoid" if block else "identity", residual_scale=0.5, eps=EPS, score_func="sigmoid",
               route_norm=True, expert_bias=c["expert_bias"], **{k: c[k] for k in names})
    announce(f"graph of an fp32 stream block={block}")
    g = MoELayerGraph(c["x"], c["w_router"], c["w13"], c["w2"], K, residual=True, **how)
    with torch.no_grad():
        for i in range(4):
            x = torch.from_numpy(rng.standard_normal((T, D)).astype(np.float32)).to(DEV)
            u, n = g(x)
            eu, en = F().moe_block(x, c["w_router"], c["w13"], c["w2"], K, **how)
            torch.cuda.synchronize()
            assert u.dtype == torch.float32 and torch.equal(u, eu), f"replay {i}"
            assert (n is None and en is None) if not block else torch.equal(n, en)


def test_graph_refuses_an_fp32_layer():
    """The layer without the block around it takes bf16 tokens."""
    MoELayerGraph = importlib.import_module("torchtitan-ascend_amd.graph").MoELayerGraph
    w13, w2 = _experts(4)
    with pytest.raises(TypeError, match="bf16"):
        MoELayerGraph(torch.zeros(2, 128), torch.zeros(4, 128, dtype=BF16), w13, w2, 2)
    with pytest.raises(TypeError, match="fp32"):
        MoELayerGraph(torch.zeros(2, 128, dtype=torch.float16), torch.zeros(4, 128, dtype=BF16), w13, w2, 2,
                      residual=True)


@pytest.mark.parametrize("only", [dict(residual_scale=0.5), dict(gate_func="sigmoid")])
def test_graph_refuses_block_arguments_without_a_block(only):
    """A scale or an activation of the gate would have nothing to act on: the
    graph would hold the bare layer and leave it out."""
    MoELayerGraph = importlib.import_module("torchtitan-ascend_amd.graph").MoELayerGraph
    w13, w2 = _experts(4)
    with pytest.raises(ValueError, match="residual"):
        MoELayerGraph(torch.zeros(2, 128, dtype=BF16), torch.zeros(4, 128, dtype=BF16), w13, w2, 2, **only)
