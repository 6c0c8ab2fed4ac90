"""The few-token layer and the 4-bit weights: what they refuse, which device their
calls run on, the module's options (CPU; nothing is launched)."""
from __future__ import annotations

import contextlib
import ctypes
import importlib
import inspect

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

BF16, F32, U8 = torch.bfloat16, torch.float32, torch.uint8
T, D, H, E, K = 6, 128, 96, 4, 2

_lib = importlib.import_module("torchtitan-ascend_amd._lib")
decode = importlib.import_module("torchtitan-ascend_amd.decode")
functional = importlib.import_module("torchtitan-ascend_amd.functional")

P16, P8 = ctypes.c_void_p(16), ctypes.c_void_p(8)
NAN = float("nan")


def err(rc):
    assert rc == 1, rc
    return _lib.load().ttamd_last_error().decode()


# ---------------------------------------------------------------------------
# C entries
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("change,want", [
    (dict(k=48), "k"), (dict(k=0), "k"), (dict(n=0), "n"), (dict(count=-1), "matrices"), (dict(w=None), "w is null"),
    (dict(w=P8), "16-byte"), (dict(codes=None), "codes is null"), (dict(exps=P8), "exponents must be 16-byte"),
    (dict(count=1 << 21), "matrices"),
])
def test_packing_refuses(change, want):
    a = dict(w=P16, count=2, n=16, k=64, codes=P16, exps=P16) | change
    lib = _lib.load()
    assert want in err(lib.ttamd_pack_e2m1(a["w"], 0, a["count"], a["n"], a["k"], a["codes"], a["exps"], None))
    if "w" not in change:
        assert want in err(lib.ttamd_unpack_e2m1(a["codes"], a["exps"], a["count"], a["n"], a["k"], a["w"], None))


@pytest.mark.parametrize("change,want", [
    (dict(E=0), "num_experts"), (dict(E=1025), "num_experts"), (dict(M=-1), "num_rows"), (dict(K=40), "k"),
    (dict(N=0), "n"), (dict(offs=None), "offs is null"), (dict(bias=P16), "bias"), (dict(x=P8), "x must be 16-byte"),
    (dict(out=None), "out is null"), (dict(codes=P8), "codes"), (dict(exps=None), "exponents"),
    (dict(M=1 << 28, N=1 << 20), "too many outputs"),
])
def test_product_refuses(change, want):
    a = dict(x=P16, codes=P16, exps=P16, offs=P16, bias=None, M=4, E=2, N=16, K=64, out=P16) | change
    assert want in err(_lib.load().ttamd_grouped_mm_e2m1(a["x"], a["codes"], a["exps"], a["offs"], a["bias"], 0, a["M"],
                                                         a["E"], a["N"], a["K"], a["out"], None))


LAYER = dict(x=P16, T=4, D=64, H=32, E=8, K=2, w_router=P16, bias=None, groups=1, kept=1, gscore=0, func=0, limit=NAN,
             w13=P16, e13=None, w2=P16, e2=None, Hs=0, s13=None, es13=None, s2=None, es2=None, gate=None, scores=P16,
             idx=P16, out=P16, ws=P16, bytes=1 << 30)
COMMON = [
    (dict(T=65), "num_tokens"), (dict(T=-1), "num_tokens"), (dict(E=0), "num_experts"), (dict(E=1025), "num_experts"),
    (dict(K=0), "topk"), (dict(K=17, E=32), "topk"), (dict(D=48), "dim"), (dict(H=40), "hidden"), (dict(H=0), "hidden"),
    (dict(Hs=-32), "shared_hidden"), (dict(Hs=48), "shared_hidden"), (dict(limit=-1.0), "swiglu_limit"),
    (dict(w13=None), "w13 is null"), (dict(w2=P8), "w2 must be 16-byte"), (dict(e13=P16), "one type"),
    (dict(e13=P16, e2=P8), "w2_exponents"), (dict(Hs=32), "w13_shared is null"),
    (dict(Hs=32, s13=P16, s2=P16, es13=P16), "experts' type"),
    (dict(Hs=32, s13=P16, s2=P16, e13=P16, e2=P16), "experts' type"), (dict(x=P8), "x must be 16-byte"),
    (dict(out=None), "out is null"), (dict(ws=None), "workspace"), (dict(bytes=64), "workspace"),
    (dict(scores=None), "null pointer"), (dict(gate=P16), "shared expert"),
    (dict(H=1 << 20, D=1 << 20, E=1024), "weights too large"),
]


def layer(change):
    a = LAYER | change
    return _lib.load().ttamd_moe_decode(
        a["x"], a["T"], a["D"], a["H"], a["E"], a["K"], a["w_router"], a["bias"], a["groups"], a["kept"], a["gscore"],
        a["func"], 0, 1e-20, 1.0, 0, a["limit"], a["w13"], a["e13"], a["w2"], a["e2"], a["Hs"], a["s13"], a["es13"],
        a["s2"], a["es2"], a["gate"], a["scores"], a["idx"], a["out"], a["ws"], a["bytes"], None)


@pytest.mark.parametrize("change,want", COMMON + [
    (dict(w_router=None), "w_router"), (dict(K=9), "topk"), (dict(groups=3), "group"), (dict(func=7), "score_func"),
    (dict(Hs=32, s13=P16, s2=P16, gate=P8), "w_gate must be 16-byte"),
])
def test_layer_refuses(change, want):
    assert want in err(layer(change))


@pytest.mark.parametrize("change,want", COMMON)
def test_expert_stage_refuses(change, want):
    a = LAYER | change
    assert want in err(_lib.load().ttamd_experts_decode(
        a["x"], a["T"], a["D"], a["H"], a["E"], a["K"], a["idx"], 1, a["scores"], 0, a["limit"], a["w13"], a["e13"],
        a["w2"], a["e2"], a["Hs"], a["s13"], a["es13"], a["s2"], a["es2"], a["gate"], a["out"], a["ws"], a["bytes"],
        None))


@pytest.mark.parametrize("change,want", [
    (dict(T=65), "num_tokens"), (dict(E=1025), "num_experts"), (dict(D=12), "dim"), (dict(K=9), "topk"),
    (dict(groups=3), "group"), (dict(func=2), "score_func"), (dict(x=None), "x is null"), (dict(w_router=P8), "w_router"),
    (dict(idx=None), "null pointer"), (dict(gate=P16), "together"), (dict(ws=P16, bytes=1), "workspace"),
])
def test_router_refuses(change, want):
    a = LAYER | change
    assert want in err(_lib.load().ttamd_router_decode(
        a["x"], a["w_router"], a["bias"], a["gate"], a["T"], a["E"], a["D"], a["K"], a["groups"], a["kept"],
        a["gscore"], a["func"], 0, 1e-20, 1.0, a["scores"], a["idx"], None, a["ws"], a["bytes"], None))


def test_calls_without_tokens_return():
    assert layer(dict(T=0, x=None, ws=None, bytes=0)) == 0
    assert _lib.load().ttamd_pack_e2m1(None, 0, 0, 16, 64, None, None, None) == 0


@pytest.mark.parametrize("D,H,K,Hs", [(32, 32, 1, 0), (2048, 768, 8, 768), (7168, 2048, 16, 2048)])
def test_workspace_of_the_largest_batch_serves_smaller_ones(D, H, K, Hs):
    lib = _lib.load()
    sizes = [lib.ttamd_experts_decode_workspace_bytes(t, D, H, K, Hs) for t in range(65)]
    whole = [lib.ttamd_moe_decode_workspace_bytes(t, D, H, 64, K, Hs) for t in range(65)]
    assert sizes == sorted(sizes) and whole == sorted(whole) and sizes[0] > 0
    assert all(w >= s for w, s in zip(whole, sizes))
    for bad in ((65, D, H, K, Hs), (-1, D, H, K, Hs), (1, 0, H, K, Hs), (1, D, H, 17, Hs), (1, D, H, K, -1)):
        assert lib.ttamd_experts_decode_workspace_bytes(*bad) == 0
    assert lib.ttamd_router_decode_workspace_bytes(-1, 8) == 0


# ---------------------------------------------------------------------------
# Python: refusals, and the device of every call
# ---------------------------------------------------------------------------
def packed(dev, e, n, k):
    u = lambda *s: torch.empty(*s, dtype=U8, device=dev)  # noqa: E731
    nb, nc = (n + 15) // 16, (k + 127) // 128
    return decode.PackedWeights(u(e, nb, nc, 64, 16), u(e, nb, (nc + 3) // 4, 64, 4), n, k)


def calls(dev):
    t = lambda *s, dtype=BF16: torch.empty(*s, dtype=dtype, device=dev)  # noqa: E731
    idx = torch.zeros(T, K, dtype=torch.int64, device=dev)
    w = (t(E, 2 * H, D), t(E, D, H))
    p = (packed(dev, E, 2 * H, D), packed(dev, E, D, H))
    s = (packed(dev, 1, 64, D), packed(dev, 1, D, 32))
    return {
        "pack_e2m1": lambda: decode.pack_e2m1(t(E, H, D)),
        "unpack_e2m1": lambda: decode.unpack_e2m1(p[0]),
        "grouped_mm_e2m1": lambda: decode.grouped_mm_e2m1(t(T, D), p[0], t(E, dtype=torch.int32)),
        "router_decode": lambda: decode.router_decode(t(T, D), t(E, D), K, shared_gate=t(1, D)),
        "experts_decode": lambda: decode.experts_decode(t(T, D), t(T, K, dtype=F32), idx, *w),
        "moe_decode": lambda: decode.moe_decode(t(T, D), t(E, D), *p, K, shared_w13=s[0], shared_w2=s[1],
                                                shared_gate=t(1, D)),
    }


class Recorder:
    def __init__(self):
        self.current, self.calls = 0, []

    def __getattr__(self, name):
        def fn(*args):
            if name.endswith("_bytes"):
                return 64
            self.calls.append((name, self.current))
            return 0

        return fn


@pytest.fixture
def recorder(monkeypatch):
    r = Recorder()
    monkeypatch.setattr(_lib, "_lib", r)
    monkeypatch.setattr(decode, "_p", lambda t: None if t is None else 256)
    monkeypatch.setattr(decode, "_stream", lambda dev: 0)
    monkeypatch.setattr(torch.Tensor, "data_ptr", lambda self: 256)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: r.current, raising=False)

    @contextlib.contextmanager
    def device(dev):
        before, r.current = r.current, dev.index
        try:
            yield
        finally:
            r.current = before

    monkeypatch.setattr(torch.cuda, "device", device)
    return r


LAUNCH = sorted(n for n, f in inspect.getmembers(decode, inspect.isfunction)
                if f.__module__ == decode.__name__ and not n.startswith("_") and n != "tile_e2m1")


@pytest.mark.parametrize("name", LAUNCH)
@pytest.mark.parametrize("index", [0, 1])
def test_calls_run_on_their_tensors_device(recorder, name, index):
    with FakeTensorMode():
        calls(torch.device("cuda", index))[name]()
    assert recorder.calls and all(dev == index for _, dev in recorder.calls), recorder.calls
    assert recorder.current == 0


def test_python_refusals(monkeypatch):
    monkeypatch.setattr(torch.Tensor, "data_ptr", lambda self: 256)
    with FakeTensorMode():
        dev = torch.device("cuda", 0)
        t = lambda *s, dtype=BF16, device=dev: torch.empty(*s, dtype=dtype, device=device)  # noqa: E731
        idx, sc = torch.zeros(T, K, dtype=torch.int64, device=dev), t(T, K, dtype=F32)
        w13, w2, p13, p2 = t(E, 2 * H, D), t(E, D, H), packed(dev, E, 2 * H, D), packed(dev, E, D, H)
        x, wr = t(T, D), t(E, D)

        def refused(kind, match, fn, *args, **kw):
            with pytest.raises(kind, match=match):
                fn(*args, **kw)

        ed, md, mm = decode.experts_decode, decode.moe_decode, decode.grouped_mm_e2m1
        refused(ValueError, "at most 64", ed, t(65, D), t(65, K, dtype=F32), idx, w13, w2)
        refused(TypeError, "int64 or int32", ed, x, sc, idx.float(), w13, w2)
        refused(ValueError, "scores and indices", ed, x, sc[:3], idx, w13, w2)
        refused(ValueError, "w13 must be", ed, x, sc, idx, w13, t(E, H, D))
        refused(TypeError, "both be bfloat16", ed, x, sc, idx, w13, p2)
        refused(TypeError, "experts' type", ed, x, sc, idx, p13, p2, shared_w13=t(64, D), shared_w2=t(D, 32))
        refused(ValueError, "together", ed, x, sc, idx, w13, w2, shared_w13=t(64, D))
        refused(ValueError, "shared_w13 must be", ed, x, sc, idx, w13, w2, shared_w13=t(64, D), shared_w2=t(D, 64))
        refused(ValueError, "shared_scale", ed, x, sc, idx, w13, w2, shared_scale=t(T, dtype=F32))
        refused(TypeError, "w13", ed, x, sc, idx, w13.float(), w2)
        refused(RuntimeError, "cuda:1", ed, x, sc, idx, w13, t(E, D, H, device="cuda:1"))
        refused(RuntimeError, "cuda:1", ed, x, sc, idx, p13, packed(torch.device("cuda", 1), E, D, H))
        refused(ValueError, "are not those", ed, x, sc, idx, p13._replace(rows=2 * H + 32), p2)
        refused(RuntimeError, "w13", ed, x, sc, idx, w13.cpu(), w2)
        refused(ValueError, "w_router", md, x, t(E + 1, D), w13, w2, K)
        refused(ValueError, "score_func", md, x, wr, w13, w2, K, "relu")
        refused(ValueError, "expert_bias", md, x, wr, w13, w2, K, expert_bias=t(E + 1, dtype=F32))
        refused(ValueError, "shared_gate needs", md, x, wr, w13, w2, K, shared_gate=t(1, D))
        refused(ValueError, "shared_gate must", md, x, wr, w13, w2, K, shared_gate=t(1, D + 8))
        refused(RuntimeError, "w_router", md, x, t(E, D, device="cuda:1"), w13, w2, K)
        refused(ValueError, "give offs", mm, x, p13)
        refused(ValueError, "x must be", mm, t(T, D + 32), p13, t(E, dtype=torch.int32))
        refused(ValueError, "offs has", mm, x, p13, t(E + 1, dtype=torch.int32))
        refused(TypeError, "offs", mm, x, p13, t(E, dtype=torch.int64))
        refused(ValueError, "bias is for", mm, x, p13, t(E, dtype=torch.int32), t(2 * H))
        refused(ValueError, "bias must be", mm, x, packed(dev, 1, H, D), None, t(H + 1))
        refused(TypeError, "uint8", mm, x, p13._replace(codes=p13.codes.float()), t(E, dtype=torch.int32))
        refused(ValueError, r"\[E, N, K\]", decode.pack_e2m1, t(D))
        refused(TypeError, "bfloat16 or float32", decode.pack_e2m1, t(E, D, dtype=torch.float16))
        refused(ValueError, "do not match", decode.tile_e2m1, t(4, 32, dtype=U8), t(4, 3, dtype=U8))
        refused(TypeError, "uint8", decode.tile_e2m1, t(4, 32), t(4, 2))
        refused(TypeError, "x must be", functional.moe_decode, x.float(), wr, w13, w2, K)
        refused(TypeError, "x must be", functional.moe_decode, x[None], wr, w13, w2, K)
        refused(ValueError, "together", functional.moe_decode, t(65, D), wr, w13, w2, K, shared_w13=t(64, D))
        refused(ValueError, "shared_gate needs", functional.moe_decode, t(65, D), wr, w13, w2, K, shared_gate=t(1, D))
        refused(TypeError, "w13 must be bfloat16", functional.moe_decode, t(65, D), wr, w13.float(), w2, K)
        # no backward
        g = lambda v: v.requires_grad_(True)  # noqa: E731
        refused(RuntimeError, "inference", ed, x, sc, idx, g(t(E, 2 * H, D)), w2)
        refused(RuntimeError, "inference", md, g(t(T, D)), wr, w13, w2, K)
        refused(RuntimeError, "inference", functional.moe_decode, g(t(65, D)), wr, w13, w2, K)
        refused(RuntimeError, "inference", mm, g(t(T, D)), packed(dev, 1, H, D))
        refused(RuntimeError, "inference", decode.pack_e2m1, g(t(E, H, D)))
        refused(RuntimeError, "inference", decode.router_decode, x, g(t(E, D)), K)


def test_cpu_tensors_have_no_fallback():
    x, wr = torch.zeros(T, D, dtype=BF16), torch.zeros(E, D, dtype=BF16)
    w13, w2 = torch.zeros(E, 2 * H, D, dtype=BF16), torch.zeros(E, D, H, dtype=BF16)
    for fn in (lambda: decode.moe_decode(x, wr, w13, w2, K), lambda: decode.router_decode(x, wr, K),
               lambda: decode.pack_e2m1(w13), lambda: functional.moe_decode(x, wr, w13, w2, K),
               lambda: decode.tile_e2m1(torch.zeros(4, 32, dtype=U8), torch.zeros(4, 2, dtype=U8))):
        with pytest.raises(RuntimeError, match="cpu|GPU|device"):
            fn()


def test_graph_refuses():
    graph = importlib.import_module("torchtitan-ascend_amd.graph")
    with FakeTensorMode():
        dev = torch.device("cuda", 0)
        t = lambda *s: torch.empty(*s, dtype=BF16, device=dev)  # noqa: E731
        x, wr, w = t(T, D), t(E, D), (t(E, 2 * H, D), t(E, D, H))
        p = (packed(dev, E, 2 * H, D), packed(dev, E, D, H))
        with pytest.raises(TypeError, match="decode=True"):
            graph.MoELayerGraph(x, wr, *p, K)
        with pytest.raises(ValueError, match="decode=True"):
            graph.MoELayerGraph(x, wr, *w, K, shared_w13=t(64, D), shared_w2=t(D, 32))
        with pytest.raises(ValueError, match="layer alone"):
            graph.MoELayerGraph(x, wr, *w, K, decode=True, residual=True)
        with pytest.raises(TypeError, match="contiguous"):
            graph.MoELayerGraph(x, wr, *w, K, decode=True, shared_w13=t(D, 64).t(), shared_w2=t(D, 32))


# ---------------------------------------------------------------------------
# The module's option
# ---------------------------------------------------------------------------
def module(pkg, **kw):
    dispatcher = pkg.HipTokenDispatcher.Config(num_experts=E, top_k=K)
    m = pkg.HipGroupedExperts.Config(dim=D, hidden_dim=H, num_experts=E, token_dispatcher=dispatcher, **kw)
    return pkg.HipGroupedExperts(m)


def test_module_packs_and_refuses_stale_copies(monkeypatch):
    pkg = importlib.import_module("torchtitan-ascend_amd")
    with pytest.raises(ValueError, match="decode_weights"):
        module(pkg, decode_weights="int4")
    with pytest.raises(RuntimeError, match="pack_weights is for"):
        module(pkg).pack_weights()
    assert module(pkg)._decode_weights() is None
    assert module(pkg, decode_weights="bf16")._decode_weights() is None  # (fp32 parameters)
    few = module(pkg, decode_weights="bf16").bfloat16()
    assert few._decode_weights()[0] is few.w13
    monkeypatch.setattr(decode, "pack_e2m1", lambda w: w.detach().clone())
    m = module(pkg, decode_weights="e2m1")
    m.init_weights()
    with pytest.raises(RuntimeError, match="call pack_weights"):
        m._decode_weights()
    m.pack_weights()
    assert torch.equal(m._decode_weights()[1], m.w2)
    with torch.no_grad():
        m.w2.mul_(2.0)
    with pytest.raises(RuntimeError, match="changed after"):
        m._decode_weights()
    m.pack_weights()
    m.load_state_dict(m.state_dict())
    with pytest.raises(RuntimeError, match="changed after"):
        m._decode_weights()
    m.pack_weights()
    m.w13 = torch.nn.Parameter(m.w13.detach().clone())
    with pytest.raises(RuntimeError, match="changed after"):
        m._decode_weights()
    m.pack_weights()
    torch.optim.SGD(m.parameters(), lr=0.1).zero_grad()
    m._decode_weights()
    for p in m.parameters():
        p.grad = torch.ones_like(p)
    torch.optim.AdamW(m.parameters(), lr=0.1).step()
    with pytest.raises(RuntimeError, match="changed after"):
        m._decode_weights()
    assert sorted(m.state_dict()) == ["w13", "w2"]


def test_converter_passes_the_option():
    pkg = importlib.import_module("torchtitan-ascend_amd")
    P = importlib.import_module("torchtitan-ascend_amd.protocol")
    for value in (None, "bf16", "e2m1"):
        mc = P.ModelConfig()
        mc.layers = [P.GroupedExperts.Config(
            dim=D, hidden_dim=H, num_experts=E,
            token_dispatcher=P.AllToAllTokenDispatcher.Config(num_experts=E, top_k=K))]
        pkg.HipGroupedExpertsConverter(pkg.HipGroupedExpertsConverter.Config(decode_weights=value)).convert(mc)
        assert mc.layers[0].decode_weights == value
    assert pkg.HipGroupedExpertsConverter.Config().decode_weights is None
