"""Recordings of the few-token operators and 4-bit weights hold their registered ops
(CPU; the C calls are stood in for, nothing is launched)."""
from __future__ import annotations

import importlib
import warnings

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

BF16, F32, U8 = torch.bfloat16, torch.float32, torch.uint8
D, H, E, K = 128, 128, 4, 2

_lib = importlib.import_module("torchtitan-ascend_amd._lib")
ops = importlib.import_module("torchtitan-ascend_amd.ops")
decode = importlib.import_module("torchtitan-ascend_amd.decode")
functional = importlib.import_module("torchtitan-ascend_amd.functional")


class Calls:
    """Stands for the library: size queries answer 64, other calls are noted."""

    def __init__(self):
        self.names = []

    def __getattr__(self, name):
        def fn(*args):
            if name.endswith("_bytes"):
                return 64
            self.names.append(name)
            return 0

        return fn


@pytest.fixture
def library(monkeypatch):
    """Ops on tensors of any device reach the recorder."""
    r = Calls()
    monkeypatch.setattr(_lib, "_lib", r)
    for m in (ops, decode):
        monkeypatch.setattr(m, "_gpu", lambda name, t: t.device)
        monkeypatch.setattr(m, "_stream", lambda dev: 0)
        monkeypatch.setattr(m, "_call", lambda dev, name, *args: getattr(r, name)(*args))
    return r


def packed(dev, e, n, k):
    codes, exps = decode._shapes(e, n, k)
    return decode.PackedWeights(torch.zeros(codes, dtype=U8, device=dev), torch.zeros(exps, dtype=U8, device=dev), n, k)


def steps(dev, tokens):
    """name -> (function of x, the ops that a recording of it has to hold)."""
    t = lambda *s, dtype=BF16: torch.zeros(*s, dtype=dtype, device=dev)  # noqa: E731
    wr, gate = t(E, D), t(1, D)
    w, s = (t(E, 2 * H, D), t(E, D, H)), (t(2 * H, D), t(D, H))
    p, q = (packed(dev, E, 2 * H, D), packed(dev, E, D, H)), (packed(dev, 1, 2 * H, D), packed(dev, 1, D, H))
    idx, scores = t(tokens, K, dtype=torch.int64), t(tokens, K, dtype=F32)
    regular = ["router", "route", "moe_experts_forward"]
    layer = ["moe_decode"] if tokens <= 64 else regular
    prompt = ["moe_decode"] if tokens <= 64 else ["router", "unpack_e2m1", "unpack_e2m1", *regular[1:], "unpack_e2m1",
                                                  "unpack_e2m1", "shared_expert_add"]
    out = {
        "layer": (lambda x: functional.moe_decode(x, wr, *w, K), layer),
        "layer_shared": (lambda x: functional.moe_decode(x, wr, *w, K, shared_w13=s[0], shared_w2=s[1],
                                                         shared_gate=gate),
                         layer if tokens <= 64 else [*regular, "shared_expert_add"]),
        "layer_packed": (lambda x: functional.moe_decode(x, wr, *p, K, shared_w13=q[0], shared_w2=q[1]), prompt),
        "product": (lambda x: functional.grouped_mm_e2m1(x, q[0], bias=t(2 * H)), ["grouped_mm_e2m1"]),
        "store": (lambda x: functional.unpack_e2m1(functional.pack_e2m1(x)), ["pack_e2m1", "unpack_e2m1"]),
    }
    if tokens <= 64:
        out["experts"] = (lambda x: functional.experts_decode(x, scores, idx, *w), ["experts_decode"])
        out["experts_packed"] = (lambda x: functional.experts_decode(x, scores, idx, *p, True, 0.5, *q),
                                 ["experts_decode"])
        out["router"] = (lambda x: functional.router_decode(x, wr, K, shared_gate=gate)[::2], ["router_decode"])
    return out


NAMES = [(n, t) for t in (9, 65) for n in steps("cpu", t)]


def recorded(graph):
    return [n.target._schema.name.split("::")[1] for n in graph.nodes
            if n.op == "call_function" and getattr(n.target, "namespace", "") == "ttamd"]


@pytest.mark.parametrize("pre_dispatch", [False, True])
@pytest.mark.parametrize("name,tokens", NAMES)
def test_make_fx_holds_the_ops(library, name, tokens, pre_dispatch):
    fn, want = steps("cpu", tokens)[name]
    with torch.no_grad():
        graph = make_fx(fn, pre_dispatch=pre_dispatch)(torch.zeros(tokens, D, dtype=BF16))
        assert recorded(graph.graph) == want
        library.names.clear()
        graph(torch.zeros(tokens, D, dtype=BF16))  # a replay makes the calls
    assert len(library.names) >= len(want)


@pytest.mark.parametrize("name,tokens", NAMES)
def test_fake_tensors_get_shapes_and_make_no_call(library, name, tokens):
    with FakeTensorMode(), torch.no_grad():
        dev = torch.device("cuda", 0)
        x = torch.zeros(tokens, D, dtype=BF16, device=dev)
        out = steps(dev, tokens)[name][0](x)
        graph = make_fx(steps(dev, tokens)[name][0])(x)
    assert not library.names
    assert recorded(graph.graph) == steps("cpu", tokens)[name][1]
    first = out[0] if isinstance(out, tuple) else out
    want = {"product": (tokens, 2 * H), "router": (tokens, K), "store": (1, tokens, D)}.get(name, (tokens, D))
    assert tuple(first.shape) == want and first.device.type == "cuda"


@pytest.mark.parametrize("name,tokens", NAMES)
def test_script_traces_hold_the_ops(library, name, tokens):
    fn, want = steps("cpu", tokens)[name]
    with torch.no_grad(), warnings.catch_warnings():
        warnings.simplefilter("ignore")  # (the batch's length becomes a constant of the trace)
        graph = torch.jit.trace(fn, (torch.zeros(tokens, D, dtype=BF16),), check_trace=False).graph
    assert [n.kind().split("::")[1] for n in graph.nodes() if n.kind().startswith("ttamd::")] == want


@pytest.mark.parametrize("name,tokens", NAMES)
def test_torch_compile_has_one_graph(library, name, tokens):
    graphs = []

    def backend(gm, inputs):
        graphs.append(gm)
        return gm.forward

    fn, want = steps("cpu", tokens)[name]
    with torch.no_grad():
        torch.compile(fn, backend=backend, fullgraph=True)(torch.zeros(tokens, D, dtype=BF16))
    torch._dynamo.reset()
    assert len(graphs) == 1
    held = [str(n.target).split(".")[1] for n in graphs[0].graph.nodes if str(n.target).startswith("ttamd.")]
    assert held == want


def test_the_modules_option_is_recorded(library):
    pkg = importlib.import_module("torchtitan-ascend_amd")
    dispatcher = pkg.HipTokenDispatcher.Config(num_experts=E, top_k=K)
    idx, scores = torch.zeros(3, 3, K, dtype=torch.int64), torch.zeros(3, 3, K)
    for option in ("bf16", "e2m1"):
        m = pkg.HipGroupedExperts(pkg.HipGroupedExperts.Config(
            dim=D, hidden_dim=H, num_experts=E, token_dispatcher=dispatcher, decode_weights=option)).bfloat16()
        if option == "e2m1":
            m.pack_weights()
        with torch.no_grad():
            graph = make_fx(lambda x: m(x, scores, idx))(torch.zeros(3, 3, D, dtype=BF16))
        assert recorded(graph.graph) == ["experts_decode"]


@pytest.mark.parametrize("choices,ops", [(16, ["experts_decode"]), (17, ["route", "moe_experts_forward"]),
                                         (64, ["route", "moe_experts_forward"])])
@pytest.mark.parametrize("option", ["bf16", "e2m1"])
def test_the_modules_option_leaves_many_choices_to_the_regular_path(library, option, choices, ops):
    """More than 16 choices a token run as they do without the option."""
    pkg = importlib.import_module("torchtitan-ascend_amd")
    dispatcher = pkg.HipTokenDispatcher.Config(num_experts=64, top_k=choices)
    m = pkg.HipGroupedExperts(pkg.HipGroupedExperts.Config(
        dim=D, hidden_dim=64, num_experts=64, token_dispatcher=dispatcher, decode_weights=option)).bfloat16()
    if option == "e2m1":
        m.pack_weights()
    idx, scores = torch.zeros(3, 3, choices, dtype=torch.int64), torch.zeros(3, 3, choices)
    with torch.no_grad():
        graph = make_fx(lambda x: m(x, scores, idx))(torch.zeros(3, 3, D, dtype=BF16))
    assert recorded(graph.graph) == ops


@pytest.mark.parametrize("tokens", [64, 65])
def test_layers_refuse_weights_on_another_device(tokens):
    """At either length, before a kernel gets their pointers."""
    with FakeTensorMode(), torch.no_grad():
        t = lambda *s, dev="cuda:0", dtype=BF16: torch.empty(*s, dtype=dtype, device=dev)  # noqa: E731
        x, good = t(tokens, D), dict(w_router=(E, D), w13=(E, 2 * H, D), w2=(E, D, H), shared_w13=(2 * H, D),
                                     shared_w2=(D, H), shared_gate=(1, D), expert_bias=(E,))
        call = functional.moe_decode if tokens > 64 else decode.moe_decode
        for dev in ("cpu", "cuda:1"):
            for name in good:
                kw = {n: t(*s, dev=dev if n == name else "cuda:0", dtype=F32 if n == "expert_bias" else BF16)
                      for n, s in good.items()}
                with pytest.raises(RuntimeError, match=name):
                    call(x, top_k=K, **kw)
            p = dict(w13=packed("cuda:0", E, 2 * H, D), w2=packed("cuda:0", E, D, H))
            for name, field in (("w13", "codes"), ("w13", "exponents"), ("w2", "codes"), ("w2", "exponents")):
                w = p[name]._replace(**{field: getattr(p[name], field).to(dev)})
                with pytest.raises(RuntimeError, match=name):
                    call(x, t(E, D), top_k=K, **(p | {name: w}))


@pytest.mark.parametrize("tokens", [9, 65])
def test_layers_take_and_refuse_the_same_forms_of_weights(library, tokens):
    t = lambda *s: torch.zeros(*s, dtype=BF16)  # noqa: E731
    x, wr, w13, w2, s13, s2 = t(tokens, D), t(1, D), t(2 * H, D), t(D, H), t(64, D), t(D, 32)
    p13, p2, q13, q2 = (packed("cpu", 1, *s) for s in ((2 * H, D), (D, H), (64, D), (D, 32)))
    with torch.no_grad():
        for w in ((w13, w2), (w13[None], w2), (p13, p2)):  # [N, K] is one expert
            shared = (q13, q2) if w[0] is p13 else (s13, s2[None])
            out = functional.moe_decode(x, wr, *w, 1, shared_w13=shared[0], shared_w2=shared[1])[0]
            assert out.shape == (tokens, D)
        for w in ((p13, w2), (w13, p2)):
            with pytest.raises(TypeError, match="both be bfloat16"):
                functional.moe_decode(x, wr, *w, 1)
        for w, shared in (((p13, p2), (s13, s2)), ((w13, w2), (q13, q2)), ((p13, p2), (q13, s2))):
            with pytest.raises(TypeError, match="experts' type"):
                functional.moe_decode(x, wr, *w, 1, shared_w13=shared[0], shared_w2=shared[1])


class Seen(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        if func.namespace == "ttamd":
            self.names.append(func._schema.name.split("::")[1])
        return func(*args, **(kwargs or {}))


class Sub(torch.Tensor):
    seen = []

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        cls.seen.append(str(func))
        return super().__torch_function__(func, types, args, kwargs or {})


def test_modes_and_subclasses_see_the_ops(library):
    x = torch.zeros(9, D, dtype=BF16)
    fn, want = steps("cpu", 9)["layer"]
    with torch.no_grad(), Seen() as mode:
        fn(x)
    assert mode.names == want
    with torch.no_grad():
        fn(x.as_subclass(Sub))
    assert any("ttamd.moe_decode" in s for s in Sub.seen)
    library.names.clear()
    with torch.no_grad():
        fn(x)  # neither: the C call at once
    assert library.names == ["ttamd_moe_decode"] and not mode.names[1:]


def direct_calls():
    wr = torch.zeros(E, D, dtype=BF16)
    w = torch.zeros(E, 2 * H, D, dtype=BF16), torch.zeros(E, D, H, dtype=BF16)
    q = packed("cpu", 1, 2 * H, D)
    idx, scores = torch.zeros(9, K, dtype=torch.int64), torch.zeros(9, K)
    return {
        "moe_decode": lambda x: decode.moe_decode(x, wr, *w, K)[0],
        "experts_decode": lambda x: decode.experts_decode(x, scores, idx, *w),
        "router_decode": lambda x: decode.router_decode(x, wr, K)[0],
        "grouped_mm_e2m1": lambda x: decode.grouped_mm_e2m1(x, q),
        "pack_e2m1": lambda x: decode.pack_e2m1(x).codes,
        "unpack_e2m1": lambda x: decode.unpack_e2m1(q),
    }


def test_direct_calls_refuse_to_be_recorded(library):
    x = torch.zeros(9, D, dtype=BF16)
    for name, fn in direct_calls().items():
        with torch.no_grad():
            for trace in (make_fx(fn), make_fx(fn, pre_dispatch=True),
                          lambda x: torch.jit.trace(fn, (x,), check_trace=False)):
                with pytest.raises(RuntimeError, match=f"functional.{name}"):
                    trace(x)
            fn(x)


@pytest.mark.parametrize("name", list(direct_calls()))
def test_direct_calls_end_a_compiled_graph(library, name):
    fn = direct_calls()[name]
    with torch.no_grad():
        out = torch.compile(lambda x: fn(x + 1).float() + 1, backend="aot_eager")(torch.zeros(9, D, dtype=BF16))
    torch._dynamo.reset()
    assert library.names == [f"ttamd_{name}"] and out.dtype == F32


@pytest.mark.parametrize("shape", [(9,), (3, 3), (1, 9), (0, 4)])
def test_fakes_have_the_shapes_of_the_calls(library, shape):
    """Rows [..., D] come back flat, traced or not."""
    t = lambda *s, dtype=BF16: torch.zeros(*s, dtype=dtype)  # noqa: E731
    wr, gate, w, q = t(E, D), t(1, D), (t(E, 2 * H, D), t(E, D, H)), packed("cpu", 1, 2 * H, D)
    idx, scores = t(*shape, K, dtype=torch.int64), t(*shape, K, dtype=F32)
    o = torch.ops.ttamd
    route = ("softmax", False, 1.0, None, 1e-20, None, None, "top2")
    fns = [lambda x: (o.experts_decode(x, scores, idx, *w, H, False, None),),
           lambda x: o.moe_decode(x, wr, *w, K, H, *route, False, None),
           lambda x: o.router_decode(x, wr, K, *route, gate),
           lambda x: (o.grouped_mm_e2m1(x, q.codes, q.exponents, 2 * H, None, None),)]
    x = t(*shape, D)
    for fn in fns:
        real = [(v.shape, v.stride(), v.dtype) for v in fn(x)]
        with FakeTensorMode(allow_non_fake_inputs=True) as mode:
            assert [(v.shape, v.stride(), v.dtype) for v in fn(mode.from_tensor(x))] == real


@pytest.mark.parametrize("experts,runs", [(256, 0), (257, 2), (300, 2), (1024, 4)])
@pytest.mark.parametrize("groups", [{}, dict(num_groups=1, topk_groups=1)])
def test_prompts_of_more_experts_than_the_fused_router_takes(library, experts, runs, groups):
    t = lambda *s: torch.zeros(*s, dtype=BF16)  # noqa: E731
    wr, w = t(experts, D), (t(experts, 2, D), t(experts, D, 1))
    with torch.no_grad():
        graph = make_fx(lambda x: functional.moe_decode(x, wr, *w, K, **groups))(t(65, D))
    routers = ["router"] * runs + ["router_topk"] if runs else ["router"]
    assert recorded(graph.graph) == [*routers, "route", "moe_experts_forward"]
    sizes = [n.args[1].meta["val"].shape[0] if runs else experts for n in graph.graph.nodes
             if str(n.target) == "ttamd.router.default"]
    assert sum(sizes) == experts and max(sizes) <= 256
