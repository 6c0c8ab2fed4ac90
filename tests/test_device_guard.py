"""Every kernel call is made with its tensors' device as the current one (CPU).

A default stream's handle is null, which the runtime takes for the current
device's: a call without the guard would run on another device than its
tensors', unordered with the calls before it.  The calls are recorded on
tensors without storage; nothing is launched."""
from __future__ import annotations

import contextlib
import importlib
import inspect

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32
T, D, H, E, K = 6, 128, 128, 4, 2
M = T * K


class Recorder:
    """Stands for the library: size queries answer 64, other calls note the
    current device and succeed."""

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
def recorder(monkeypatch, ops):
    r = Recorder()
    monkeypatch.setattr(ops._lib, "_lib", r)
    monkeypatch.setattr(ops, "_p", lambda t: None if t is None else 256)
    monkeypatch.setattr(ops, "_stream", lambda dev: 0)
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


def calls(ops, dev):
    """One call of every public function of ops that launches kernels."""
    t = lambda *s, dtype=BF16: torch.empty(*s, dtype=dtype, device=dev)  # noqa: E731
    f, i, u = (lambda *s, d=d: t(*s, dtype=d) for d in (F32, I32, torch.uint8))
    i64 = lambda *s: t(*s, dtype=torch.int64)  # noqa: E731
    routing = ops.RouteResult(i(E), i(E + 1), i(M), i(M), f(M), None)
    packed = lambda rows, cols: ops.PackedRows(u(rows, cols), u(rows, (cols + 127) // 128))  # noqa: E731
    xq, sx = u(M, D), f(D // 128, M)
    return {
        "router_topk": lambda: ops.router_topk(f(T, E), K),
        "router_topk_backward": lambda: ops.router_topk_backward(f(T, K), i64(T, K), f(T, E)),
        "router_fused": lambda: ops.router_fused(t(T, D), t(E, D), K),
        "router_backward": lambda: ops.router_backward(f(T, K), i64(T, K), t(T, E), t(T, D), t(E, D)),
        "router_route": lambda: ops.router_route(t(T, D), t(E, D), K),
        "experts_forward": lambda: ops.experts_forward(t(T, D), routing, t(E, 2 * H, D), t(E, D, H), K, False),
        "route": lambda: ops.route(i64(T, K), E, f(T, K)),
        "gather_rows": lambda: ops.gather_rows(t(T, D), i(M), K),
        "permute_rows": lambda: ops.permute_rows(t(T, D), routing, K),
        "dispatch_rows": lambda: ops.dispatch_rows(t(T, D), i(M), K),
        "gather_rows_exact": lambda: ops.gather_rows_exact(t(T, D), i(T)),
        "scatter_rows_exact": lambda: ops.scatter_rows_exact(t(T, D), i(T)),
        "token_permute": lambda: ops.token_permute(t(T, D), i64(T, K), E),
        "token_unpermute": lambda: ops.token_unpermute(t(M, D), i(M), f(M), K),
        "token_unpermute_grad": lambda: ops.token_unpermute_grad(t(T, D), i(M), f(M), t(M, D), K, True),
        "combine": lambda: ops.combine(t(M, D), i(M), f(M), K),
        "rowdot_scatter": lambda: ops.rowdot_scatter(t(M, D), t(T, D), i(M), K),
        "sum_topk": lambda: ops.sum_topk(t(M, D), K),
        "residual_norm": lambda: ops.residual_norm(t(T, D), t(T, D), pre_weight=t(D)),
        "rms_norm": lambda: ops.rms_norm(t(T, D), t(D)),
        "combine_norm": lambda: ops.combine_norm(t(M, D), K, residual=t(T, D)),
        "residual_norm_backward": lambda: ops.residual_norm_backward(t(T, D), None, t(T, D), f(2, T), t(T, D)),
        "group_labels": lambda: ops.group_labels(i(2, E), E, M),
        "grouped_mm": lambda: ops.grouped_mm(t(M, D), t(E, H, D), i(E)),
        "grouped_mm_swiglu": lambda: ops.grouped_mm_swiglu(t(M, D), t(E, 2 * H, D), i(E)),
        "grouped_mm_swiglu_gather": lambda: ops.grouped_mm_swiglu_gather(t(T, D), i(M), K, t(E, 2 * H, D), i(E)),
        "grouped_mm_unpermute": lambda: ops.grouped_mm_unpermute(t(M, H), t(E, D, H), i(E)),
        "grouped_mm_dgrad": lambda: ops.grouped_mm_dgrad(t(M, H), t(E, H, D), i(E)),
        "grouped_mm_dgrad_swiglu": lambda: ops.grouped_mm_dgrad_swiglu(t(M, D), t(E, D, H), t(M, 2 * H), i(E)),
        "grouped_mm_wgrad": lambda: ops.grouped_mm_wgrad(t(M, D), t(M, H), i(E), E),
        "pack_e4m3": lambda: ops.pack_e4m3(t(T, D)),
        "unpack_e4m3": lambda: ops.unpack_e4m3(packed(T, D)),
        "grouped_mm_dgrad_swiglu_packed": lambda: ops.grouped_mm_dgrad_swiglu_packed(
            t(M, D), t(E, D, H), packed(M, 2 * H), i(E)),
        "grouped_mm_wgrad_packed": lambda: ops.grouped_mm_wgrad_packed(t(M, H), packed(T, D), i(E), E, src_index=i(M),
                                                                       src_div=K),
        "shared_expert_add": lambda: ops.shared_expert_add(t(T, D), t(T, D), t(2 * H, D), t(D, H)),
        "quantize_fp8_rows": lambda: ops.quantize_fp8_rows(t(M, D)),
        "quantize_fp8_blocks": lambda: ops.quantize_fp8_blocks(t(E, H, D)),
        "grouped_mm_fp8": lambda: ops.grouped_mm_fp8(xq, sx, u(E, H, D), f(E, H // 128, D // 128), i(E)),
        "grouped_mm_fp8_swiglu": lambda: ops.grouped_mm_fp8_swiglu(
            xq, sx, u(E, 2 * H, D), f(E, 2 * H // 128, D // 128), i(E)),
        "grouped_mm_fp8_unpermute": lambda: ops.grouped_mm_fp8_unpermute(xq, sx, u(E, H, D), f(E, H // 128, D // 128),
                                                                         i(E)),
    }


# not kernel launches: host queries and the timing probes
HOST = {"gemm_tiles", "probe_next_gemm", "probe_launches"}


def names():
    ops = importlib.import_module("torchtitan-ascend_amd.ops")
    return sorted(n for n, f in inspect.getmembers(ops, inspect.isfunction)
                  if f.__module__ == ops.__name__ and not n.startswith("_") and n not in HOST)


@pytest.mark.parametrize("name", names())
@pytest.mark.parametrize("index", [0, 1])
def test_calls_run_on_their_tensors_device(recorder, ops, name, index):
    with FakeTensorMode():
        calls(ops, torch.device("cuda", index))[name]()
    assert recorder.calls and all(dev == index for _, dev in recorder.calls), recorder.calls
    assert recorder.current == 0


def test_graph_is_captured_on_its_tensors_device(recorder, ops, monkeypatch):
    """MoELayerGraph of tensors on another device than the current one: warm-up,
    capture and the calls in them."""
    graph = importlib.import_module("torchtitan-ascend_amd.graph")
    captured = []

    class Stream:
        def __init__(self, device=None):
            self.device = device

        def wait_stream(self, other):
            pass

    @contextlib.contextmanager
    def capture(_graph, stream=None):
        # (torch's default capture stream belongs to the first device it was used on)
        captured.append((recorder.current, stream.device.index))
        yield

    monkeypatch.setattr(torch.cuda, "Stream", Stream)
    monkeypatch.setattr(torch.cuda, "stream", lambda s: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_stream", lambda dev=None: Stream(dev))
    monkeypatch.setattr(torch.cuda, "CUDAGraph", lambda: None)
    monkeypatch.setattr(torch.cuda, "graph", capture)
    with FakeTensorMode():
        t = lambda *s: torch.empty(*s, dtype=BF16, device="cuda:1")  # noqa: E731
        graph.MoELayerGraph(t(T, D), t(E, D), t(E, 2 * H, D), t(E, D, H), K)
    assert captured == [(1, 1)]
    assert recorder.calls and all(dev == 1 for _, dev in recorder.calls)
    assert recorder.current == 0
