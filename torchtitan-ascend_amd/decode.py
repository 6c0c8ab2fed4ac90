"""The MoE layer for a few tokens (a decode batch), and 4-bit weights.

A batch of at most 64 tokens streams the weights of the experts it hits once
and computes almost nothing with them, so it takes other kernels than the
grouped GEMMs of `ops`: `moe_decode` is the whole layer (router, experts,
combine, shared expert), `experts_decode` its expert stage on given picks, both
with bf16 or 4-bit weights; `pack_e2m1` makes the latter, `grouped_mm_e2m1`
multiplies a few rows with them.  For serving: none has a backward, and a call
under autograd with a tensor that requires a gradient raises.

Like `ops`, every function allocates with torch's caching allocator and calls
the C ABI on torch's current stream of its tensors' device; there is no
fallback.  A tracer sees nothing of such a call, so the functions refuse to run under
one; those of the same names in `functional` take the registered ops there.
Reference: NpuGroupedExperts.forward with its router
(torchtitanturbo/models/common/npu_gmm.py:100-110; models/qwen3_5/model.py:752-809).
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib, ops
from .ops import _call, _gpu, _groups, _limit, _p, _same_device, _stream, _want

_BF16 = torch.bfloat16
_U8 = torch.uint8
MAX_TOKENS = 64
MAX_TOPK = 16


class PackedWeights(NamedTuple):
    """Weights [E, N, K] (or [N, K] as E = 1) in 4 bits: e2m1 codes with one
    power-of-two scale per row and 32 columns, value = code * 2^(exponent - 127),
    exact in bf16 (tile layout: ttamd_pack_e2m1)."""

    codes: torch.Tensor  # uint8 [E, ceil(N / 16), ceil(K / 128), 64, 16]
    exponents: torch.Tensor  # uint8 [E, ceil(N / 16), ceil(K / 512), 64, 4]
    rows: int  # N
    cols: int  # K


_tracing, _mode = torch._C._is_tracing, torch._C._get_dispatch_mode
_included, _mode_count = torch._C._dispatch_tls_is_dispatch_key_included, torch._C._len_torch_dispatch_stack
_PRE_DISPATCH, _PROXY = torch._C.DispatchKey.PreDispatch, torch._C._TorchDispatchModeKey.PROXY


def _seen() -> bool:
    """Whether a tracer or another dispatch mode is at work."""
    return _mode_count() > 0 or _tracing() or _included(_PRE_DISPATCH)


def _no_grad(name: str, *tensors) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and type(t) is not PackedWeights and getattr(t, "requires_grad", False):
                raise RuntimeError(f"{name} is for inference (it has no backward); call it under torch.no_grad()")


def _direct(name: str, *tensors) -> None:
    """Refuse a call under torch.jit.trace or make_fx, whose recording would hold the
    outputs' allocation and not the kernels, and one that asks for gradients."""
    if torch.compiler.is_dynamo_compiling():
        pass  # (the graph ends in front of the C call)
    elif (_mode_count() or _tracing() or _included(_PRE_DISPATCH)) and (
            _tracing() or _included(_PRE_DISPATCH) or _mode(_PROXY) is not None):
        raise RuntimeError(f"decode.{name} cannot be recorded by a tracer: call functional.{name}")
    _no_grad(name, *tensors)


def _shapes(E: int, N: int, K: int) -> tuple[tuple, tuple]:
    nb, nc = (N + 15) // 16, (K + 127) // 128
    return (E, nb, nc, 64, 16), (E, nb, (nc + 3) // 4, 64, 4)


# (device and dtype comparisons written out here and below: a call on one token is
# bound by the host, and keyword helpers take half a microsecond each)
def _packed(name: str, w: PackedWeights, dev: torch.device) -> tuple[torch.Tensor, torch.Tensor, int]:
    """(codes, exponents, E) of packed weights, checked."""
    codes, exps, N, K = w
    if codes.dtype is not _U8 or exps.dtype is not _U8:
        raise TypeError(f"{name}: codes and exponents must be uint8, got {codes.dtype} and {exps.dtype}")
    if codes.device != dev or exps.device != dev:
        raise RuntimeError(f"{name} is on {codes.device} and {exps.device}, expected {dev}")
    E = codes.shape[0] if codes.dim() == 5 else 0
    nb, nc = (N + 15) // 16, (K + 127) // 128
    if N < 1 or K < 1 or codes.shape != (E, nb, nc, 64, 16) or exps.shape != (E, nb, (nc + 3) // 4, 64, 4):
        raise ValueError(f"{name}: codes {tuple(codes.shape)} and exponents {tuple(exps.shape)} are not those of "
                         f"[E, {N}, {K}] weights")
    return codes.contiguous(), exps.contiguous(), E


def pack_e2m1(w: torch.Tensor) -> PackedWeights:
    """4-bit form of weights w [E, N, K] or [N, K], bf16 or fp32, K % 32 == 0
    (ttamd_pack_e2m1): 17/32 byte per value, each within a quarter of its
    magnitude, or within 2^-2 of a 32-column group's scale where that is more.
    A group that holds a NaN or an infinity becomes NaN."""
    dev = _gpu("w", w)
    _direct("pack_e2m1", w)
    if w.dim() not in (2, 3):
        raise ValueError(f"w must be [E, N, K] or [N, K], got {tuple(w.shape)}")
    if w.dtype not in (_BF16, torch.float32):
        raise TypeError(f"w must be bfloat16 or float32, got {w.dtype}")
    w = w.contiguous()
    E, (N, K) = (w.shape[0] if w.dim() == 3 else 1), w.shape[-2:]
    codes_shape, exps_shape = _shapes(E, N, K)
    codes, exps = w.new_empty(codes_shape, dtype=_U8), w.new_empty(exps_shape, dtype=_U8)
    _call(dev, "ttamd_pack_e2m1", w.data_ptr(), 1 if w.dtype is torch.float32 else 0, E, N, K, codes.data_ptr(),
          exps.data_ptr(), _stream(dev))
    return PackedWeights(codes, exps, N, K)


def unpack_e2m1(w: PackedWeights) -> torch.Tensor:
    """The bf16 values [E, N, K] of packed weights, exactly (ttamd_unpack_e2m1):
    for prompts, whose rows fill the grouped GEMMs."""
    dev = _gpu("w.codes", w.codes)
    _direct("unpack_e2m1")
    codes, exps, E = _packed("w", w, dev)
    out = codes.new_empty((E, w.rows, w.cols), dtype=_BF16)
    _call(dev, "ttamd_unpack_e2m1", codes.data_ptr(), exps.data_ptr(), E, w.rows, w.cols, out.data_ptr(),
          _stream(dev))
    return out


def tile_e2m1(codes: torch.Tensor, exponents: torch.Tensor) -> PackedWeights:
    """PackedWeights from row-major 4-bit weights, as checkpoints hold them: codes
    uint8 [..., N, K / 2], two to a byte, the even column in the low half, and
    exponent bytes uint8 [..., N, K / 32] (value = code * 2^(byte - 127)).  A
    re-ordering by torch operations, done once when weights are loaded."""
    dev = _gpu("codes", codes)
    _same_device(dev, exponents=exponents)
    if codes.dtype != torch.uint8 or exponents.dtype != torch.uint8:
        raise TypeError("codes and exponents must be uint8")
    if codes.dim() not in (2, 3) or codes.shape[-1] % 16 or \
            tuple(exponents.shape) != (*codes.shape[:-1], codes.shape[-1] // 16):
        raise ValueError(f"codes [..., N, K / 2] {tuple(codes.shape)} and exponents [..., N, K / 32] "
                         f"{tuple(exponents.shape)} do not match")
    N, K = codes.shape[-2], 2 * codes.shape[-1]
    E = codes.shape[0] if codes.dim() == 3 else 1
    (_, nb, nc, _, _), exps_shape = _shapes(E, N, K)
    pad = torch.nn.functional.pad
    c = pad(codes.reshape(E, N, K // 2), (0, nc * 64 - K // 2, 0, nb * 16 - N))
    c = c.view(E, nb, 16, nc, 4, 16).permute(0, 1, 3, 4, 2, 5).reshape(E, nb, nc, 64, 16).contiguous()
    x = pad(exponents.reshape(E, N, K // 32), (0, 16 * exps_shape[2] - K // 32, 0, nb * 16 - N), value=127)
    x = x.view(E, nb, 16, exps_shape[2], 4, 4).permute(0, 1, 3, 5, 2, 4).reshape(exps_shape).contiguous()
    return PackedWeights(c, x, N, K)


def grouped_mm_e2m1(
    x: torch.Tensor, w: PackedWeights, offs: torch.Tensor | None = None, bias: torch.Tensor | None = None
) -> torch.Tensor:
    """out[m] = x[m] @ w[e]^T (+ bias) with 4-bit weights (ttamd_grouped_mm_e2m1):
    x bf16 [M, K] (without offs also [..., K]); expert e's rows end at offs[e]
    (int32 [E]) as in grouped_mm, or all rows take the one matrix of w.  bias [N]
    bf16 or fp32, without offs.  For few rows: an expert with more rows than a pass
    holds (4 to 64, by the average) reads its weights again, so a prompt takes
    unpack_e2m1 and a matrix product.  Rows at or past offs[-1] are not written."""
    dev = _gpu("x", x)
    _direct("grouped_mm_e2m1", x, bias)
    x = _want("x", x, _BF16)
    codes, exps, E = _packed("w", w, dev)
    N, K = w.rows, w.cols
    shape = x.shape
    if shape[-1] != K or (offs is not None and len(shape) != 2):
        raise ValueError(f"x must be [M, {K}], got {tuple(shape)}")
    if offs is None:
        if E != 1:
            raise ValueError(f"w holds {E} matrices: give offs")
    else:
        _same_device(dev, offs=offs)
        offs = _want("offs", offs, torch.int32)
        if offs.numel() != E:
            raise ValueError(f"offs has {offs.numel()} entries, w holds {E} matrices")
        if bias is not None:
            raise ValueError("bias is for a call without offs")
    if bias is not None:
        _same_device(dev, bias=bias)
        if bias.dtype not in (_BF16, torch.float32) or bias.numel() != N:
            raise ValueError(f"bias must be [{N}], bfloat16 or float32")
        bias = bias.contiguous()
    out = x.new_empty((*shape[:-1], N))
    _call(dev, "ttamd_grouped_mm_e2m1", x.data_ptr(), codes.data_ptr(), exps.data_ptr(), _p(offs), _p(bias),
          1 if bias is not None and bias.dtype is torch.float32 else 0, x.numel() // K, E, N, K, out.data_ptr(),
          _stream(dev))
    return out


def _rows(x: torch.Tensor) -> torch.Tensor:
    x = _want("x", x if x.dim() == 2 else x.reshape(-1, x.shape[-1]), _BF16)
    if x.shape[0] > MAX_TOKENS:
        raise ValueError(f"at most {MAX_TOKENS} tokens, got {x.shape[0]}: a longer batch fills the grouped GEMMs "
                         "(functional.moe_decode chooses)")
    return x


def _bias(expert_bias: torch.Tensor | None, E: int, dev: torch.device) -> torch.Tensor | None:
    if expert_bias is None:
        return None
    _same_device(dev, expert_bias=expert_bias)
    expert_bias = expert_bias.float().contiguous()
    if expert_bias.shape != (E,):
        raise ValueError("expert_bias must be [E]")
    return expert_bias


def _gate_row(shared_gate: torch.Tensor | None, D: int, dev: torch.device) -> torch.Tensor | None:
    if shared_gate is None:
        return None
    _same_device(dev, shared_gate=shared_gate)
    shared_gate = _want("shared_gate", shared_gate, _BF16)
    if shared_gate.numel() != D:
        raise ValueError(f"shared_gate must be [1, {D}], got {tuple(shared_gate.shape)}")
    return shared_gate


def _weight(name: str, w, dev: torch.device) -> tuple[torch.Tensor, torch.Tensor | None, tuple]:
    """(tensor, exponents or None, (E, N, K)) of bf16 [E, N, K] / [N, K] or packed weights."""
    if isinstance(w, PackedWeights):
        codes, exps, E = _packed(name, w, dev)
        return codes, exps, (E, w.rows, w.cols)
    if w.device != dev:
        _gpu(name, w)
        raise RuntimeError(f"{name} is on {w.device}, expected {dev}")
    w = _want(name, w, _BF16)
    shape = w.shape
    if len(shape) == 3:
        return w, None, shape
    if len(shape) != 2:
        raise ValueError(f"{name} must be [E, N, K], got {tuple(shape)}")
    return w, None, (1, *shape)


def _experts(w13, w2, shared_w13, shared_w2, D: int, dev: torch.device):
    """(E, H, Hs, the data pointers of the eight weight tensors, the tensors) of the layer's weights, checked."""
    t13, e13, s13 = _weight("w13", w13, dev)
    t2, e2, s2 = _weight("w2", w2, dev)
    E, H = s13[0], s13[1] // 2
    if s13[2] != D or s13[1] % 2 or tuple(s2) != (E, D, H):
        raise ValueError(f"w13 must be [E, 2H, {D}] and w2 [E, {D}, H]; got {tuple(s13)}, {tuple(s2)}")
    if (e13 is None) != (e2 is None):
        raise TypeError("w13 and w2 must both be bfloat16 or both packed")
    keep = (t13, e13, t2, e2)
    if shared_w13 is None and shared_w2 is None:
        return E, H, 0, (t13.data_ptr(), _p(e13), t2.data_ptr(), _p(e2)), (None, None, None, None), keep
    if shared_w13 is None or shared_w2 is None:
        raise ValueError("give shared_w13 and shared_w2 together")
    u13, f13, z13 = _weight("shared_w13", shared_w13, dev)
    u2, f2, z2 = _weight("shared_w2", shared_w2, dev)
    Hs = z13[1] // 2
    if z13[0] != 1 or z13[2] != D or z13[1] % 2 or tuple(z2) != (1, D, Hs):
        raise ValueError(f"shared_w13 must be [2Hs, {D}] and shared_w2 [{D}, Hs]; got {tuple(z13)}, {tuple(z2)}")
    if (f13 is None) != (e13 is None) or (f2 is None) != (e13 is None):
        raise TypeError("the shared expert's weights must be of the experts' type")
    return (E, H, Hs, (t13.data_ptr(), _p(e13), t2.data_ptr(), _p(e2)),
            (u13.data_ptr(), _p(f13), u2.data_ptr(), _p(f2)), (*keep, u13, f13, u2, f2))


def router_decode(
    x: torch.Tensor,
    w_router: torch.Tensor,
    top_k: int,
    score_func: str = "softmax",
    route_norm: bool = False,
    route_scale: float = 1.0,
    expert_bias: torch.Tensor | None = None,
    norm_eps: float = 1e-20,
    num_groups: int | None = None,
    topk_groups: int | None = None,
    group_score: str = "top2",
    shared_gate: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """Router of at most 64 tokens (ttamd_router_decode): (top_scores fp32 [T, K],
    selected_experts_indices int64 [T, K], gate fp32 [T] or None).  Arguments as
    ops.router_fused; the bf16 logits come from 64-bit sums and the selection is
    ops.router_topk's with groups (one group without num_groups).  shared_gate [1,
    D] bf16: gate = sigmoid of the token's bf16 product with it."""
    dev = _gpu("x", x)
    _direct("router_decode", x, w_router, shared_gate)
    x = _rows(x)
    w_router = _want("w_router", w_router, _BF16)
    _same_device(dev, w_router=w_router)
    T, D = x.shape
    E = w_router.shape[0]
    if w_router.dim() != 2 or w_router.shape[1] != D:
        raise ValueError(f"w_router must be [E, {D}], got {tuple(w_router.shape)}")
    if score_func not in ops._SCORE_FUNCS:
        raise ValueError(f"score_func must be one of {sorted(ops._SCORE_FUNCS)}")
    groups = _groups(num_groups, topk_groups, group_score) or (1, 1, 0)
    expert_bias = _bias(expert_bias, E, dev)
    shared_gate = _gate_row(shared_gate, D, dev)
    scores = torch.empty(T, top_k, dtype=torch.float32, device=dev)
    idx = torch.empty(T, top_k, dtype=torch.int64, device=dev)
    gate = None if shared_gate is None else torch.empty(T, dtype=torch.float32, device=dev)
    ws = torch.empty(max(16, _lib.load().ttamd_router_decode_workspace_bytes(T, E)), dtype=_U8, device=dev)
    _call(dev, "ttamd_router_decode", _p(x), _p(w_router), _p(expert_bias), _p(shared_gate), T, E, D, top_k, *groups,
          ops._SCORE_FUNCS[score_func], int(bool(route_norm)), float(norm_eps), float(route_scale), _p(scores), _p(idx),
          _p(gate), _p(ws), ws.numel(), _stream(dev))
    return scores, idx, gate


def experts_decode(
    x: torch.Tensor,
    top_scores: torch.Tensor,
    selected_experts_indices: torch.Tensor,
    w13: torch.Tensor | PackedWeights,
    w2: torch.Tensor | PackedWeights,
    score_before_experts: bool = False,
    swiglu_limit: float | None = None,
    shared_w13: torch.Tensor | PackedWeights | None = None,
    shared_w2: torch.Tensor | PackedWeights | None = None,
    shared_scale: torch.Tensor | None = None,
) -> torch.Tensor:
    """Expert stage of at most 64 tokens on given picks (ttamd_experts_decode): x bf16
    [T, D], scores and indices [T, K] (int64 or int32; one outside [0, E) adds
    nothing) -> bf16 [T, D].  Weights bf16 (w13 [E, 2H, D], w2 [E, D, H]) or all
    packed.  A shared expert [2Hs, D] / [D, Hs] is added times shared_scale fp32 [T]
    (None: 1)."""
    dev = _gpu("x", x)
    _direct("experts_decode", x, top_scores, w13, w2, shared_w13, shared_w2, shared_scale)
    x = _rows(x)
    T, D = x.shape
    idx = selected_experts_indices
    if idx.dtype not in (torch.int64, torch.int32):
        raise TypeError("expert indices must be int64 or int32")
    K = idx.shape[-1]
    _same_device(dev, top_scores=top_scores, selected_experts_indices=idx, shared_scale=shared_scale)
    if idx.numel() != T * K or top_scores.numel() != T * K:
        raise ValueError(f"scores and indices must be [{T}, K], got {tuple(top_scores.shape)} and {tuple(idx.shape)}")
    idx, top_scores = idx.contiguous(), top_scores.float().contiguous()
    E, H, Hs, weights, shared, _keep = _experts(w13, w2, shared_w13, shared_w2, D, dev)
    if shared_scale is not None:
        shared_scale = shared_scale.float().contiguous()
        if Hs == 0 or shared_scale.numel() != T:
            raise ValueError(f"shared_scale must be [{T}] and needs a shared expert")
    lib = _lib._lib or _lib.load()
    out = x.new_empty((T, D))
    ws = x.new_empty(lib.ttamd_experts_decode_workspace_bytes(T, D, H, K, Hs), dtype=_U8)
    _call(dev, "ttamd_experts_decode", x.data_ptr(), T, D, H, E, K, idx.data_ptr(),
          1 if idx.dtype is torch.int64 else 0, top_scores.data_ptr(), 1 if score_before_experts else 0,
          _limit(swiglu_limit), *weights, Hs, *shared, _p(shared_scale), out.data_ptr(), ws.data_ptr(), ws.numel(),
          _stream(dev))
    return out


def moe_decode(
    x: torch.Tensor,
    w_router: torch.Tensor,
    w13: torch.Tensor | PackedWeights,
    w2: torch.Tensor | PackedWeights,
    top_k: int,
    score_func: str = "softmax",
    route_norm: bool = False,
    route_scale: float = 1.0,
    expert_bias: torch.Tensor | None = None,
    norm_eps: float = 1e-20,
    num_groups: int | None = None,
    topk_groups: int | None = None,
    group_score: str = "top2",
    score_before_experts: bool = False,
    swiglu_limit: float | None = None,
    shared_w13: torch.Tensor | PackedWeights | None = None,
    shared_w2: torch.Tensor | PackedWeights | None = None,
    shared_gate: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The MoE layer of at most 64 tokens in one call (ttamd_moe_decode): x bf16
    [T, D] to (out bf16 [T, D], top_scores fp32 [T, K], selected_experts_indices
    int64 [T, K]).  Router arguments as router_decode, expert arguments as
    experts_decode; shared_gate [1, D] scales the shared expert by sigmoid(x .
    shared_gate)."""
    dev = _gpu("x", x)
    _direct("moe_decode", x, w_router, w13, w2, shared_w13, shared_w2, shared_gate)
    x = _rows(x)
    T, D = x.shape
    E, H, Hs, weights, shared, _keep = _experts(w13, w2, shared_w13, shared_w2, D, dev)
    w_router = _want("w_router", w_router, _BF16)
    if w_router.device != dev:
        raise RuntimeError(f"w_router is on {w_router.device}, expected {dev}")
    if w_router.shape != (E, D):
        raise ValueError(f"w_router must be [{E}, {D}] for these experts, got {tuple(w_router.shape)}")
    func = ops._SCORE_FUNCS.get(score_func)
    if func is None:
        raise ValueError(f"score_func must be one of {sorted(ops._SCORE_FUNCS)}")
    groups = _groups(num_groups, topk_groups, group_score) or (1, 1, 0)
    if expert_bias is not None:
        expert_bias = _bias(expert_bias, E, dev)
    if shared_gate is not None:
        shared_gate = _gate_row(shared_gate, D, dev)
        if Hs == 0:
            raise ValueError("shared_gate needs a shared expert")
    lib = _lib._lib or _lib.load()
    scores = x.new_empty((T, top_k), dtype=torch.float32)
    idx = x.new_empty((T, top_k), dtype=torch.int64)
    out = x.new_empty((T, D))
    ws = x.new_empty(lib.ttamd_moe_decode_workspace_bytes(T, D, H, E, top_k, Hs), dtype=_U8)
    _call(dev, "ttamd_moe_decode", x.data_ptr(), T, D, H, E, top_k, w_router.data_ptr(), _p(expert_bias), *groups,
          func, 1 if route_norm else 0, norm_eps, route_scale, 1 if score_before_experts else 0, _limit(swiglu_limit),
          *weights, Hs, *shared, _p(shared_gate), scores.data_ptr(), idx.data_ptr(), out.data_ptr(), ws.data_ptr(),
          ws.numel(), _stream(dev))
    return out, scores, idx
