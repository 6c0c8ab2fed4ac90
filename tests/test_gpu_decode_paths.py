"""The few-token operators as the framework uses them: captured and replayed, on
other streams and beside each other, through the module, the serving layer and the
registered ops; what a value that is not finite reaches; the ends of the sizes.

Bounds: test_gpu_decode.py.  Where two forms run the same kernels on the same values
the comparison is bit for bit."""
from __future__ import annotations

import importlib

import numpy as np
import pytest
import torch

from gpu_util import DEV, announce
from test_gpu_decode import BF16, build, check_product, layer_ref, weights

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def decode():
    return importlib.import_module("torchtitan-ascend_amd.decode")


@pytest.fixture(scope="module")
def functional():
    return importlib.import_module("torchtitan-ascend_amd.functional")


def layer(decode, rng, T, E, D, H, bits, shared):
    w, wb = build(decode, rng, E, D, H, bits, shared)
    x, wr, wg = weights(rng, T, D, scale=1.0), weights(rng, E, D), weights(rng, 1, D)
    kw = dict(shared_w13=w[2], shared_w2=w[3], shared_gate=wg) if shared else {}
    return x, wr, w[:2], kw, wb


# ---------------------------------------------------------------------------
# Graphs and streams
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("T,E,K,D,H,shared", [(1, 16, 2, 256, 128, 0), (7, 8, 2, 160, 96, 64), (64, 8, 2, 512, 288, 96),
                                              (33, 40, 4, 96, 64, 0)])
@pytest.mark.parametrize("bits", [16, 4])
def test_graph_replays_equal_eager(decode, T, E, K, D, H, shared, bits):
    graph = importlib.import_module("torchtitan-ascend_amd.graph")
    rng = np.random.default_rng(T)
    x, wr, w, kw, _ = layer(decode, rng, T, E, D, H, bits, shared)
    announce(f"graph decode T={T} E={E} bits={bits}")
    g = graph.MoELayerGraph(x, wr, *w, K, "sigmoid", True, decode=True, **kw)
    for i in range(5):
        xi = weights(rng, T, D, scale=1.0 + i)
        got = g(xi).clone()
        want = decode.moe_decode(xi, wr, *w, K, "sigmoid", True, **kw)[0]
        assert torch.equal(got, want), i
        torch.cuda.synchronize()
        assert torch.equal(g(xi), want), i
    with torch.no_grad():  # weights are read in place
        (w[0].codes if bits == 4 else w[0]).copy_((w[0].codes if bits == 4 else w[0]).flip(0))
    want = decode.moe_decode(xi, wr, *w, K, "sigmoid", True, **kw)[0]
    assert torch.equal(g.replay(), want)


def test_two_graphs_of_one_pool(decode):
    """Captured one after the other into a shared pool, replayed in that order."""
    rng = np.random.default_rng(2)
    a = layer(decode, rng, 16, 8, 256, 128, 4, 96)
    b = layer(decode, rng, 64, 32, 128, 64, 16, 0)
    runs = [lambda: decode.moe_decode(a[0], a[1], *a[2], 2, **a[3])[0],
            lambda: decode.moe_decode(b[0], b[1], *b[2], 4)[0]]
    want = [r() for r in runs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    announce("two graphs, one pool")
    for r in runs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side, pool=graphs[0].pool() if graphs else None):
            outs.append(r())
        graphs.append(g)
    for _ in range(4):
        for o in outs:
            o.zero_()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
        runs[1](), runs[0]()


def test_streams_beside_each_other(decode):
    """Two layers and a product in flight on three streams."""
    rng = np.random.default_rng(3)
    a = layer(decode, rng, 64, 16, 512, 256, 4, 0)
    b = layer(decode, rng, 5, 64, 512, 256, 16, 64)
    pw = decode.pack_e2m1(weights(rng, 1000, 1440))
    px = weights(rng, 13, 1440, scale=1.0)
    runs = [lambda: decode.moe_decode(a[0], a[1], *a[2], 2)[0],
            lambda: decode.moe_decode(b[0], b[1], *b[2], 6, **b[3])[0],
            lambda: decode.grouped_mm_e2m1(px, pw)]
    want = [r() for r in runs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in runs]
    announce("three streams")
    for _ in range(3):
        got = []
        for _ in range(8):
            for s, r in zip(streams, runs):
                with torch.cuda.stream(s):
                    got.append(r())
        torch.cuda.synchronize()
        for i, y in enumerate(got):
            assert torch.equal(y, want[i % 3]), i


# ---------------------------------------------------------------------------
# The framework's own paths
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("T", [1, 64, 65, 200])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("shared", [0, 128])
def test_serving_layer_of_any_length(decode, functional, T, bits, shared):
    rng = np.random.default_rng(T + bits)
    E, K, D, H = 8, 2, 256, 128
    x, wr, w, kw, wb = layer(decode, rng, T, E, D, H, bits, shared)
    announce(f"functional.moe_decode T={T} bits={bits} shared={shared}")
    out, s, i = functional.moe_decode(x, wr, *w, K, "softmax", True, swiglu_limit=0.7, **kw)
    if T <= 64:
        want = decode.moe_decode(x, wr, *w, K, "softmax", True, swiglu_limit=0.7, **kw)
        assert torch.equal(out, want[0]) and torch.equal(s, want[1]) and torch.equal(i, want[2])
        return
    with torch.no_grad():
        s2, i2 = functional.router(x, wr, K, "softmax", True)
        want = functional.moe_experts_forward(x, s2, i2, *wb[:2], E, False, 0.7)
        if shared:
            want = functional.shared_expert_combine(want, x, *wb[2:], x @ kw["shared_gate"][0], 0.7)
    assert torch.equal(s, s2) and torch.equal(i, i2) and torch.equal(out, want)


@pytest.mark.parametrize("score_before", [False, True])
@pytest.mark.parametrize("T", [(1, 1), (4, 16), (5, 13)])
def test_module_option(decode, functional, T, score_before):
    """HipGroupedExperts: 64 tokens and fewer without autograd take the streams, others
    and the default the path they took."""
    pkg = importlib.import_module("torchtitan-ascend_amd")
    E, K, D, H = 8, 2, 256, 128
    rng = np.random.default_rng(T[1])
    tokens = T[0] * T[1]
    idx = torch.from_numpy(np.argsort(rng.random((*T, E)), axis=-1)[..., :K].copy()).to(DEV)
    scores, x = torch.rand(*T, K, device=DEV), weights(rng, *T, D, scale=1.0)
    out = {}
    for option in (None, "bf16", "e2m1"):
        dispatcher = pkg.HipTokenDispatcher.Config(num_experts=E, top_k=K, score_before_experts=score_before)
        m = pkg.HipGroupedExperts(pkg.HipGroupedExperts.Config(
            dim=D, hidden_dim=H, num_experts=E, token_dispatcher=dispatcher, swiglu_limit=0.9,
            decode_weights=option)).to(DEV).bfloat16()
        with torch.no_grad():
            m.w13.copy_(weights(np.random.default_rng(1), E, 2 * H, D))
            m.w2.copy_(weights(np.random.default_rng(2), E, D, H))
        if option == "e2m1":
            m.pack_weights()
        announce(f"module {option} {tokens}")
        with torch.no_grad():
            out[option] = m(x, scores, idx)
        # autograd: the path of every batch
        y = m(x, scores, idx)
        y.sum().backward()
        assert m.w13.grad is not None and (option is None or torch.equal(y, train))
        train = y.detach()
    flat = (x.view(tokens, D), scores.view(tokens, K), idx.view(tokens, K))
    w13, w2 = m.w13.detach(), m.w2.detach()
    with torch.no_grad():
        plain = functional.moe_experts_forward(*flat, w13, w2, E, score_before, 0.9)
        packed = [decode.pack_e2m1(w) for w in (w13, w2)]
        few = {o: plain if tokens > 64 else decode.experts_decode(*flat, *w, score_before, 0.9)
               for o, w in (("bf16", (w13, w2)), ("e2m1", packed))}
    assert torch.equal(out[None].view(tokens, D), plain)
    for option, want in few.items():
        assert torch.equal(out[option].view(tokens, D), want), option


def _op_cases(decode):
    rng = np.random.default_rng(8)
    T, E, K, D, H, Hs = 6, 4, 2, 128, 96, 64
    x, wr, wg = weights(rng, T, D, scale=1.0), weights(rng, E, D), weights(rng, 1, D)
    full, _ = build(decode, np.random.default_rng(9), E, D, H, 16, Hs)
    p = [decode.pack_e2m1(w) for w in full]
    idx = torch.from_numpy(np.argsort(rng.random((T, E)), axis=1)[:, :K].copy()).to(DEV)
    scores = torch.rand(T, K, device=DEV)
    ops = torch.ops.ttamd
    offs = torch.tensor([2, 2, 5, 6], dtype=torch.int32, device=DEV)
    route = ("softmax", True, 1.0, None, 1e-20, None, None, "top2", False, None)
    return {
        "product": (ops.grouped_mm_e2m1, (x, p[0].codes, p[0].exponents, 2 * H, offs, None)),
        "product_bias": (ops.grouped_mm_e2m1, (x.view(2, 3, D), p[2].codes, p[2].exponents, 2 * Hs, None,
                                               torch.rand(2 * Hs, device=DEV))),
        "experts": (ops.experts_decode, (x, scores, idx, *full[:2], H, False, None)),
        "experts_packed": (ops.experts_decode, (
            x, scores, idx, p[0].codes, p[1].codes, H, True, 0.5, p[0].exponents, p[1].exponents, Hs, p[2].codes,
            p[3].codes, p[2].exponents, p[3].exponents, torch.rand(T, device=DEV))),
        "layer": (ops.moe_decode, (x, wr, *full[:2], K, H, *route)),
        "layer_packed": (ops.moe_decode, (
            x, wr, p[0].codes, p[1].codes, K, H, *route, p[0].exponents, p[1].exponents, Hs, p[2].codes, p[3].codes,
            p[2].exponents, p[3].exponents, wg)),
    }


@pytest.mark.parametrize("name", ["product", "product_bias", "experts", "experts_packed", "layer", "layer_packed"])
def test_opcheck(decode, name):
    importlib.import_module("torchtitan-ascend_amd.library")
    op, args = _op_cases(decode)[name]
    announce(f"opcheck {name}")
    torch.library.opcheck(op, args)


@pytest.mark.parametrize("bits", [16, 4])
def test_under_torch_compile(decode, functional, bits):
    rng = np.random.default_rng(4)
    x, wr, w, kw, _ = layer(decode, rng, 9, 8, 128, 64, bits, 96)

    @torch.compile(backend="aot_eager", fullgraph=True)
    def step(x, w, kw):
        out, scores, idx = functional.moe_decode(x, wr, *w, 2, **kw)
        return out + functional.experts_decode(out, scores, idx, *w), scores, idx

    with torch.no_grad():
        got = step(x, w, kw)
        out, scores, idx = decode.moe_decode(x, wr, *w, 2, **kw)
        want = out + decode.experts_decode(out, scores, idx, *w)
    assert torch.equal(got[0], want) and torch.equal(got[1], scores) and torch.equal(got[2], idx)


# ---------------------------------------------------------------------------
# Values that are not finite
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("T", [4, 24, 64])
@pytest.mark.parametrize("bits", [16, 4])
def test_values_that_are_not_finite_stay_in_their_rows(decode, T, bits):
    """A NaN or an infinity in a token reaches that token's output only; one in an
    expert's weights the tokens that chose it; in another expert's, nothing."""
    rng = np.random.default_rng(T)
    E, K, D, H = 6, 2, 160, 96  # (rows that end inside a stage)
    w, _ = build(decode, rng, E, D, H, 16)
    w = [t.clone() for t in w]
    x = weights(rng, T, D, scale=1.0)
    idx = torch.from_numpy(np.argsort(rng.random((T, E - 1)), axis=1)[:, :K].copy()).to(DEV)  # nobody takes expert 5
    scores = torch.rand(T, K, device=DEV)
    form = (lambda ts: [decode.pack_e2m1(t) for t in ts]) if bits == 4 else (lambda ts: ts)
    clean = decode.experts_decode(x, scores, idx, *form(w))
    assert torch.isfinite(clean).all()
    w[0][5], w[1][5] = float("nan"), float("inf")
    announce(f"non-finite T={T} bits={bits}")
    assert torch.equal(decode.experts_decode(x, scores, idx, *form(w)), clean)
    xs = x.clone()
    xs[1, D - 1] = float("nan")
    xs[3, 0] = float("inf")
    y = decode.experts_decode(xs, scores, idx, *form(w))
    rest = [t for t in range(T) if t not in (1, 3)]
    assert torch.isnan(y[1]).all() and torch.equal(y[rest], clean[rest])
    assert not torch.isfinite(y[3]).all()
    w[1][2, 7, H - 1] = float("nan")
    y = decode.experts_decode(x, scores, idx, *form(w))
    took = (idx == 2).any(1)
    assert torch.isnan(y[took, 7]).all() and torch.equal(y[~took], clean[~took])
    keep = [d for d in range(D) if d != 7]
    assert torch.equal(y[:, keep], clean[:, keep])


@pytest.mark.parametrize("M", [2, 20, 40])
def test_products_keep_values_that_are_not_finite_in_their_rows(decode, M):
    rng = np.random.default_rng(M)
    N, K = 50, 288
    w, x = weights(rng, N, K), weights(rng, M, K, scale=1.0)
    clean = decode.grouped_mm_e2m1(x, decode.pack_e2m1(w))
    xs, ws = x.clone(), w.clone()
    xs[1, K - 1], ws[49, 3] = float("inf"), float("nan")
    y = decode.grouped_mm_e2m1(xs, decode.pack_e2m1(ws))
    assert torch.isnan(y[:, 49]).all() and not torch.isfinite(y[1]).any()
    rest = [m for m in range(M) if m != 1]
    assert torch.equal(y[rest][:, :49], clean[rest][:, :49])


# ---------------------------------------------------------------------------
# Sizes, strides, batches
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("T,E,K,D,H,shared", [
    (64, 1024, 16, 32, 32, 0), (64, 512, 16, 64, 32, 32), (64, 256, 16, 160, 32, 0), (64, 16, 16, 96, 64, 0),
    (1, 2, 2, 16384, 64, 0), (4, 2, 1, 64, 8192, 32), (64, 1, 1, 8192, 32, 0), (16, 700, 10, 32, 96, 0),
    (20, 20, 5, 4128, 32, 0), (8, 3, 1, 4352, 160, 0), (63, 12, 2, 6400, 64, 32),
])
def test_ends_of_the_sizes(decode, T, E, K, D, H, shared, bits):
    rng = np.random.default_rng(T + E + D)
    w, wb = build(decode, rng, E, D, H, bits, shared)
    x = weights(rng, T, D, scale=1.0)
    idx = torch.from_numpy(np.argsort(rng.random((T, E)), axis=1)[:, :K].copy()).to(DEV)
    scores = torch.rand(T, K, device=DEV)
    announce(f"ends T={T} E={E} K={K} D={D} H={H} Hs={shared} bits={bits}")
    y = decode.experts_decode(x, scores, idx, *w[:2], False, None, *(w[2:] or (None, None)))
    ref, bound = layer_ref(x, scores, idx, *wb[:2], False, None, wb[2:] or None)
    off = ((y.double() - ref).abs() - bound).max().item()
    assert off <= 0, f"{off:.3e} past the bound"


@pytest.mark.parametrize("M", [1, 16, 17, 33, 64, 65, 200])
def test_dense_product_over_the_row_tiles(decode, M):
    rng = np.random.default_rng(M)
    x, p = weights(rng, M, 544, scale=1.0), decode.pack_e2m1(weights(rng, 75, 544))
    announce(f"rows {M}")
    y = decode.grouped_mm_e2m1(x, p)
    check_product(x, decode.unpack_e2m1(p)[0], y)
    assert torch.equal(decode.grouped_mm_e2m1(x.view(1, M, 544), p), y[None])


def gpu_weights(seed, *shape):
    g = torch.Generator(DEV).manual_seed(seed)
    return torch.randn(*shape, device=DEV, dtype=BF16, generator=g) * 0.05


@pytest.mark.parametrize("E,N,K,counts", [(40, 4096, 4096, 20), (33, 2048, 4224, 36)])
def test_grouped_product_with_a_short_last_round(decode, E, N, K, counts):
    """More runs than whole rounds of the chip, long rows: the last ones are shared."""
    x, p = gpu_weights(1, E * counts, K) * 20, decode.pack_e2m1(gpu_weights(2, E, N, K))
    offs = torch.arange(1, E + 1, dtype=torch.int32, device=DEV) * counts
    announce(f"last round E={E} N={N} K={K}")
    y = decode.grouped_mm_e2m1(x, p, offs)
    w = decode.unpack_e2m1(p)
    for e in range(E):
        rows = slice(e * counts, (e + 1) * counts)
        check_product(x[rows], w[e], y[rows])


@pytest.mark.parametrize("T,E,K,D,H,Hs", [(64, 32, 2, 4096, 1024, 256), (40, 36, 8, 4096, 1024, 0)])
def test_layer_with_a_short_last_round(decode, T, E, K, D, H, Hs):
    pairs = [gpu_weights(3, E, 2 * H, D), gpu_weights(4, E, D, H)]
    pairs += [gpu_weights(5, 2 * Hs, D), gpu_weights(6, D, Hs)] if Hs else []
    w = [decode.pack_e2m1(t) for t in pairs]
    wb = [decode.unpack_e2m1(p).view(t.shape) for p, t in zip(w, pairs)]
    x = gpu_weights(7, T, D) * 20
    idx = (torch.arange(T * K, device=DEV) % E).view(T, K)
    scores = torch.rand(T, K, device=DEV)
    announce(f"layer, last round T={T} E={E}")
    y = decode.experts_decode(x, scores, idx, *w[:2], False, 0.9, *(w[2:] or (None, None)))
    ref, bound = layer_ref(x, scores, idx, *wb[:2], False, 0.9, wb[2:] or None)
    off = ((y.double() - ref).abs() - bound).max().item()
    assert off <= 0, f"{off:.3e} past the bound"


def test_offsets_out_of_order_stay_in_bounds(decode):
    """Ends that fall, pass the rows or are negative leave rows unwritten; nothing
    outside the rows is touched."""
    rng = np.random.default_rng(0)
    p = decode.pack_e2m1(weights(rng, 5, 48, 96))
    x = weights(rng, 12, 96, scale=1.0)
    offs = torch.tensor([-3, 4, 2, 99, 99], dtype=torch.int32, device=DEV)
    y = decode.grouped_mm_e2m1(x, p, offs)
    w = decode.unpack_e2m1(p)
    check_product(x[:2], w[1], y[:2])  # rows 2 and 3: of two experts
    check_product(x[4:], w[3], y[4:])


@pytest.mark.parametrize("bits", [16, 4])
def test_strides_and_views(decode, bits):
    """Rows of a wider buffer, transposed picks, weights that are views."""
    rng = np.random.default_rng(6)
    T, E, K, D, H = 10, 5, 2, 128, 64
    w, _ = build(decode, rng, E, D, H, bits)
    wide = weights(rng, T, 2 * D, scale=1.0)
    idx = torch.from_numpy(np.argsort(rng.random((T, E)), axis=1)[:, :K].copy()).to(DEV)
    scores = torch.rand(K, T, device=DEV).t()
    y = decode.experts_decode(wide[:, D:], scores, idx.t().contiguous().t(), *w)
    assert torch.equal(y, decode.experts_decode(wide[:, D:].contiguous(), scores.contiguous(), idx, *w))
    assert torch.equal(y, decode.experts_decode(wide[:, D:], scores.double(), idx.int(), *w))
    if bits == 16:
        view = torch.cat([w[0], w[0]], 2)[:, :, :D]
        assert torch.equal(y, decode.experts_decode(wide[:, D:], scores, idx, view, w[1]))
    else:
        some = decode.PackedWeights(torch.stack([w[0].codes] * 2, 1)[:, 0], w[0].exponents, 2 * H, D)
        assert torch.equal(y, decode.experts_decode(wide[:, D:], scores, idx, some, w[1]))


@pytest.mark.parametrize("bits", [16, 4])
def test_padded_batch(decode, bits):
    """Rows of a padded batch whose labels name no expert: zeros, and the others as if
    they were not there."""
    rng = np.random.default_rng(12)
    E, K, D, H, real = 8, 2, 256, 96, 11
    w, wb = build(decode, rng, E, D, H, bits)
    x = weights(rng, 32, D, scale=1.0)
    x[real:] = float("nan")
    idx = torch.from_numpy(np.argsort(rng.random((32, E)), axis=1)[:, :K].copy()).to(DEV)
    idx[real:] = -1
    scores = torch.rand(32, K, device=DEV)
    scores[real:] = float("nan")
    y = decode.experts_decode(x, scores, idx, *w)
    assert not y[real:].any()
    ref, bound = layer_ref(x[:real], scores[:real], idx[:real], *wb, False, None)
    assert ((y[:real].double() - ref).abs() - bound).max() <= 0


def test_a_serving_step(decode, functional):
    """Together, as they would be used: 4-bit weights from a prompt's pass to single
    tokens, a projection and the layer per step, captured."""
    rng = np.random.default_rng(21)
    E, K, D, H = 16, 4, 256, 128
    x, wr, w, kw, wb = layer(decode, rng, 96, E, D, H, 4, 128)
    proj = decode.pack_e2m1(weights(rng, D, D))
    prompt = functional.moe_decode(x, wr, *w, K, **kw)[0]
    assert torch.isfinite(prompt).all()

    def step(h):
        out = decode.moe_decode(decode.grouped_mm_e2m1(h, proj), wr, *w, K, **kw)
        return (h + out[0], *out)

    last = x[-4:].clone()
    h = last.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.no_grad(), torch.cuda.stream(side):
        step(h)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        nxt, out, s, i = step(h)
    announce("serving step")
    for n in range(4):
        h.copy_(last)
        g.replay()
        want = step(last)
        assert torch.equal(nxt, want[0]) and torch.equal(i, want[3])
        z = decode.grouped_mm_e2m1(last, proj)
        gate = decode.router_decode(z, wr, K, shared_gate=kw["shared_gate"])[2]
        ref, bound = layer_ref(z, s, i, *wb[:2], False, None, wb[2:], gate)
        assert ((out.double() - ref).abs() - bound).max() <= 0, n
        last = want[0]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("picks", [[3, 3, 1, 3], [-1, 2, 4, 1], [4, 9, -7, 2 ** 33], [0, 1, 2, 3]])
@pytest.mark.parametrize("shared", [0, 64])
def test_one_token_of_any_picks(decode, bits, picks, shared):
    """Repeated picks and picks of no expert, none left at all."""
    rng = np.random.default_rng(31)
    E, D, H = 4, 288, 160
    w, wb = build(decode, rng, E, D, H, bits, shared)
    x, scores = weights(rng, 1, D, scale=1.0), torch.rand(1, 4, device=DEV)
    idx = torch.tensor([picks], device=DEV)
    scale = torch.rand(1, device=DEV) if shared else None
    announce(f"one token {picks} bits={bits} shared={shared}")
    y = decode.experts_decode(x, scores, idx, *w[:2], False, None, *(w[2:] or (None, None)), scale)
    ref, bound = layer_ref(x, scores, idx, *wb[:2], False, None, wb[2:] or None, scale)
    assert ((y.double() - ref).abs() - bound).max() <= 0


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("E,K,kw", [
    (1, 1, {}), (256, 8, {}), (257, 8, {}), (128, 9, {}), (60, 4, dict(score_func="sigmoid", route_norm=True)),
    (64, 6, dict(num_groups=8, topk_groups=3)), (96, 8, dict(num_groups=4, topk_groups=2, group_score="max")),
    (16, 2, dict(score_before_experts=True, swiglu_limit=0.5))])
@pytest.mark.parametrize("biased", [False, True])
def test_one_token_of_any_router(decode, ops, bits, E, K, kw, biased):
    """The selection made with the first product against the router's own, and both
    forms of the expert stage against each other."""
    rng = np.random.default_rng(E + K)
    D, H = 160, 64
    x, wr, w, shared, _ = layer(decode, rng, 1, E, D, H, bits, 32)
    kw = dict(kw, expert_bias=torch.randn(E, device=DEV) * 0.1) if biased else kw
    route = {k: v for k, v in kw.items() if k not in ("score_before_experts", "swiglu_limit")}
    announce(f"one token E={E} K={K} {kw.keys()} bits={bits}")
    out, s, i = decode.moe_decode(x, wr, *w, K, **kw, **shared)
    s2, i2, gate = decode.router_decode(x, wr, K, shared_gate=shared["shared_gate"], **route)
    assert torch.equal(s, s2) and torch.equal(i, i2)
    want = decode.experts_decode(x, s2, i2, *w, kw.get("score_before_experts", False), kw.get("swiglu_limit"),
                                 shared["shared_w13"], shared["shared_w2"], gate)
    assert torch.equal(out, want)
    # the same token twice: the plan's kernel instead
    both = decode.moe_decode(x.expand(2, -1), wr, *w, K, **kw, **shared)
    assert torch.equal(both[1], s.expand(2, -1)) and torch.equal(both[2], i.expand(2, -1))


@pytest.mark.parametrize("option", ["bf16", "e2m1"])
def test_module_option_under_torch_compile(option):
    pkg = importlib.import_module("torchtitan-ascend_amd")
    E, K, D, H = 8, 2, 256, 128
    rng = np.random.default_rng(5)
    dispatcher = pkg.HipTokenDispatcher.Config(num_experts=E, top_k=K)
    m = pkg.HipGroupedExperts(pkg.HipGroupedExperts.Config(
        dim=D, hidden_dim=H, num_experts=E, token_dispatcher=dispatcher, decode_weights=option)).to(DEV).bfloat16()
    m.init_weights()
    if option == "e2m1":
        m.pack_weights()
    idx = torch.from_numpy(np.argsort(rng.random((2, 9, E)), axis=-1)[..., :K].copy()).to(DEV)
    scores, x = torch.rand(2, 9, K, device=DEV), weights(rng, 2, 9, D, scale=1.0)
    announce(f"compiled module {option}")
    with torch.no_grad():
        want = m(x, scores, idx)
        # (the check that the 4-bit copies are of the present parameters breaks the graph)
        assert torch.equal(torch.compile(m, backend="aot_eager", fullgraph=option == "bf16")(x, scores, idx), want)


@pytest.mark.parametrize("T", [1, 5, 64])
@pytest.mark.parametrize("bits", [16, 4])
def test_weights_past_32_bits(decode, T, bits):
    """Experts that lie 5 GB apart give what they give side by side."""
    E, K, D, H = (40, 2, 8192, 4096) if bits == 16 else (80, 2, 16384, 4096)
    g = torch.Generator(DEV).manual_seed(T)
    if bits == 16:
        w = [torch.empty(E, 2 * H, D, dtype=BF16, device=DEV), torch.empty(E, D, H, dtype=BF16, device=DEV)]
    else:
        w = [decode.PackedWeights(torch.empty(c, dtype=torch.uint8, device=DEV),
                                  torch.empty(e, dtype=torch.uint8, device=DEV), n, k)
             for n, k in ((2 * H, D), (D, H)) for c, e in (decode._shapes(E, n, k),)]
        assert w[0].codes.numel() > 2 ** 32
    at = [0, E // 2, E - 1]
    for t in w:
        for e in at:
            if bits == 16:
                t[e] = torch.randn(t.shape[1:], generator=g, device=DEV) * 0.02
            else:
                t.codes[e] = torch.randint(0, 256, t.codes.shape[1:], generator=g, device=DEV, dtype=torch.uint8)
                t.exponents[e] = 120
    if bits == 16:
        near = [t[at].clone() for t in w]
        assert w[0].numel() * 2 > 2 ** 32
    else:
        near = [decode.PackedWeights(t.codes[at].clone(), t.exponents[at].clone(), t.rows, t.cols) for t in w]
    x = torch.randn(T, D, generator=g, device=DEV).to(BF16)
    idx = torch.stack([torch.arange(T, device=DEV) % 3, (torch.arange(T, device=DEV) + 2) % 3], 1)
    scores = torch.rand(T, K, device=DEV)
    announce(f"past 32 bits T={T} bits={bits}")
    pad = torch.tensor(at, device=DEV)
    y = decode.experts_decode(x, scores, pad[idx], *w)
    z = decode.experts_decode(x, scores, idx, *near)
    ref, bound = layer_ref(x, scores, idx, *(near if bits == 16 else map(decode.unpack_e2m1, near)), False, None)
    for got in (y, z):  # (not the same bits: the choice of kernels goes by tokens per expert)
        assert ((got.double() - ref).abs() - bound).max() <= 0


@pytest.mark.parametrize("option", [None, "bf16"])
def test_module_without_tokens(option):
    pkg = importlib.import_module("torchtitan-ascend_amd")
    m = pkg.HipGroupedExperts(pkg.HipGroupedExperts.Config(
        dim=128, hidden_dim=128, num_experts=4, decode_weights=option,
        token_dispatcher=pkg.HipTokenDispatcher.Config(num_experts=4, top_k=2))).to(DEV).bfloat16()
    m.init_weights()
    with torch.no_grad():
        y = m(torch.empty(0, 3, 128, dtype=BF16, device=DEV), torch.empty(0, 3, 2, device=DEV),
              torch.empty(0, 3, 2, dtype=torch.int64, device=DEV))
    assert y.shape == (0, 128)
