"""The inference MoE layer forward captured as one HIP graph.

A step of the layer is two C-ABI calls (ttamd_router_route, then
ttamd_moe_experts_forward: six kernel launches, all on the caller's
stream, none of them a memset, a host synchronisation or an allocation
inside the library).  At small shapes the host's cost per call exceeds
the kernels' run time (the debug shape: T = 2048, D = 256), so the pair
is recorded once with torch's graph capture over that stream and replayed:
one launch per step.  Every buffer the step uses (the routing outputs, the
tile plan, the workspaces, the output) is allocated once, during capture,
from the graph's private pool.

Reference: the step is NpuGroupedExperts.forward with its router
(torchtitanturbo/models/common/npu_gmm.py:100-110; router closed form
models/qwen3_5/model.py:752-766), inference only.
"""
from __future__ import annotations

import torch

from . import decode as _few
from . import ops
from .functional import moe_block

_BF16 = torch.bfloat16


class MoELayerGraph:
    """Router + dispatch + experts + combine for a fixed [T, D] input shape,
    captured once and replayed.

    ``layer(x)`` copies x into the graph's input buffer, replays the graph
    on the current stream and returns the graph's output buffer: the next
    call overwrites it, so clone it to keep it.  Weights are read where they
    are at capture time (update them in place, not by rebinding).

    With ``residual``, or any of the norm weights or a gate, the graph holds
    the block around the layer (functional.moe_block: norm, layer, norm, gate,
    residual sum, next norm; the gate is read in place too) and returns (u, n);
    x, the residual stream, is then bf16 or fp32.

    With ``decode`` the step is decode.moe_decode (at most 64 tokens): its weights may
    be packed in 4 bits, and it takes a shared expert.
    """

    def __init__(
        self,
        x: torch.Tensor,
        w_router: torch.Tensor,
        w13: torch.Tensor,
        w2: torch.Tensor,
        top_k: int,
        score_func: str = "softmax",
        route_norm: bool = False,
        score_before_experts: bool = False,
        route_scale: float = 1.0,
        expert_bias: torch.Tensor | None = None,
        swiglu_limit: float | None = None,
        warmup: int = 2,
        num_groups: int | None = None,
        topk_groups: int | None = None,
        group_score: str = "top2",
        pre_weight: torch.Tensor | None = None,
        post_weight: torch.Tensor | None = None,
        gate: torch.Tensor | None = None,
        gate_func: str = "identity",
        residual_scale: float = 1.0,
        next_weight: torch.Tensor | None = None,
        eps: float = 1e-6,
        residual: bool = False,
        decode: bool = False,
        shared_w13: torch.Tensor | _few.PackedWeights | None = None,
        shared_w2: torch.Tensor | _few.PackedWeights | None = None,
        shared_gate: torch.Tensor | None = None,
    ):
        block = residual or any(t is not None for t in (pre_weight, post_weight, gate, next_weight))
        if x.dim() != 2 or x.dtype != _BF16 and not (block and x.dtype == torch.float32):
            raise TypeError("x must be a bf16 [T, D] tensor, or an fp32 one with the block around the layer")
        if not block and (residual_scale != 1.0 or gate_func != "identity"):
            raise ValueError("residual_scale and gate_func need the block: residual=True, a norm weight or a gate")
        shared = (shared_w13, shared_w2, shared_gate)
        if decode and block:
            raise ValueError("decode is for the layer alone, without the block around it")
        if not decode and any(t is not None for t in shared):
            raise ValueError("a shared expert needs decode=True")
        for name, t in zip(("w_router", "w13", "w2", "shared_w13", "shared_w2", "shared_gate"),
                           (w_router, w13, w2, *shared)):
            if isinstance(t, _few.PackedWeights):
                if not decode:
                    raise TypeError(f"{name}: 4-bit weights need decode=True")
                if not (t.codes.is_contiguous() and t.exponents.is_contiguous()):
                    raise TypeError(f"{name} must be contiguous (read in place by the graph)")
            elif t is not None and (t.dtype != _BF16 or not t.is_contiguous()):
                raise TypeError(f"{name} must be a contiguous bf16 tensor (read in place by the graph)")
        self._shared = dict(zip(("shared_w13", "shared_w2", "shared_gate"), shared)) if decode else None
        self._args = (w_router, w13, w2, top_k, score_func, route_norm, score_before_experts, route_scale,
                      expert_bias, swiglu_limit)
        self._groups = dict(num_groups=num_groups, topk_groups=topk_groups, group_score=group_score)
        self._block = None
        if block:
            self._block = dict(pre_weight=pre_weight, post_weight=post_weight, gate=gate, gate_func=gate_func,
                               residual_scale=residual_scale, next_weight=next_weight, eps=eps)
        self.static_x = x.detach().clone()
        # warm up on a side stream (first calls set kernel attributes), then capture
        side = torch.cuda.Stream(device=x.device)
        side.wait_stream(torch.cuda.current_stream(x.device))
        with torch.no_grad(), torch.cuda.stream(side):
            for _ in range(warmup):
                self._step(self.static_x)
        torch.cuda.current_stream(x.device).wait_stream(side)
        self.graph = torch.cuda.CUDAGraph()
        with torch.no_grad(), torch.cuda.device(x.device), torch.cuda.graph(self.graph, stream=side):
            self.static_out = self._step(self.static_x)

    def _step(self, x: torch.Tensor):
        w_router, w13, w2, top_k, func, norm, before, scale, bias, limit = self._args
        if self._block is not None:
            return moe_block(x, w_router, w13, w2, top_k, score_func=func, route_norm=norm, route_scale=scale,
                             expert_bias=bias, score_before_experts=before, swiglu_limit=limit, **self._block,
                             **self._groups)
        if self._shared is not None:
            return _few.moe_decode(x, w_router, w13, w2, top_k, func, norm, scale, bias, score_before_experts=before,
                                   swiglu_limit=limit, **self._groups, **self._shared)[0]
        _, _, r = ops.router_route(x, w_router, top_k, func, norm, scale, bias, with_inverse=False,
                                    **self._groups)
        return ops.experts_forward(x, r, w13, w2, top_k, before, limit)

    def __call__(self, x: torch.Tensor):
        if x.shape != self.static_x.shape:
            raise ValueError(f"captured for x {tuple(self.static_x.shape)}, got {tuple(x.shape)}")
        self.static_x.copy_(x)
        self.graph.replay()
        return self.static_out

    def replay(self):
        """Replay on the input already in ``static_x``."""
        self.graph.replay()
        return self.static_out
