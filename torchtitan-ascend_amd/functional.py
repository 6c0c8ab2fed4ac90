"""Autograd-carrying functions of the MoE expert path (HIP kernels forward
and backward), built on the registered ``ttamd::*`` custom ops of
``library.py`` so that torch.compile / AOTAutograd trace them as opaque
nodes with their registered backward.

The split follows the reference's module boundaries so each piece can be used
on its own:

  router    (UPSTREAM TokenChoiceTopKRouter; closed form qwen3_5/model.py:752-766)
  dispatch  (upstream dispatch, entered from npu_gmm.py:106-108)
      routed[j] = x[s_j // K] (* score[s_j] when score_before_experts)
  experts   (_run_experts_grouped_mm, npu_gmm.py:21-40)
      y = grouped_mm(swiglu(clamp(grouped_mm(routed, w13))), w2)
  combine   (upstream combine, npu_gmm.py:110)
      out[t] = sum_k (score[t,k] if score after experts else 1) * y[pos(t,k)]

plus the reference's own NPUMoeTokenUnpermute (npu_permute.py:15-53), the
norms around the block (models/common/npu_rmsnorm.py:15-37) and `moe_block`,
the whole of them.
`moe_experts_forward` chains them; without autograd it takes the fused
inference op (one C-ABI call for the whole expert stage).  `moe_decode` is a
serving step's layer, `experts_decode` its expert stage for a few tokens.
"""
from __future__ import annotations

import torch

from . import decode
from . import library  # noqa: F401  (registers the ttamd::* ops)
from . import ops
from .decode import PackedWeights

_BF16 = torch.bfloat16
_T = torch.ops.ttamd


def _bf16(w: torch.Tensor) -> torch.Tensor:
    return library._bf(w)


def _needs_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def router(
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
) -> tuple[torch.Tensor, torch.Tensor]:
    """UPSTREAM TokenChoiceTopKRouter forward: (top_scores fp32 [T, K],
    selected_experts_indices int64 [T, K]).  x [..., D] and w_router [E, D]
    in any float dtype (bf16 inside the op, so their gradients come back in
    their own dtype); differentiable in x and w_router through ttamd::router's
    registered backward, the expert ids carry no gradient.  num_groups and
    topk_groups limit a token's experts to its topk_groups best of num_groups
    equal runs of experts (see ops.router_topk)."""
    xb = x.reshape(-1, x.shape[-1]).to(_BF16).contiguous()
    scores, idx, _ = _T.router(xb, w_router, top_k, score_func, route_norm, route_scale, expert_bias, norm_eps,
                               num_groups, topk_groups, group_score)
    return scores, idx


def router_topk(
    logits: torch.Tensor,
    top_k: int,
    score_func: str = "softmax",
    route_norm: bool = False,
    route_scale: float = 1.0,
    expert_bias: torch.Tensor | None = None,
    norm_eps: float = 1e-20,
    num_groups: int | None = None,
    topk_groups: int | None = None,
    group_score: str = "top2",
) -> tuple[torch.Tensor, torch.Tensor]:
    """The router's selection from given logits [T, E], differentiable in them
    (models/qwen3_5/model.py:757-765): (top_scores fp32 [T, K],
    selected_experts_indices int64 [T, K]); arguments as ops.router_topk."""
    return _T.router_topk(logits, top_k, score_func, route_norm, route_scale, expert_bias, norm_eps, num_groups,
                          topk_groups, group_score)


def dispatch(x, scores_flat, sorted_indices, inverse, sorted_scores, top_k, score_before):
    """routed = gather of token rows in stable expert order (+ score before experts)."""
    return _T.dispatch(x, scores_flat, sorted_indices, inverse, sorted_scores, top_k, score_before)


def experts(routed, w13, w2, offs, swiglu_limit):
    """y = (swiglu(clamp(x @ w13[e]^T))) @ w2[e]^T over ragged expert groups;
    the pre-activation, the SwiGLU output and (for weights that are not bf16)
    the forward's bf16 weight copies are kept only when a backward can
    follow."""
    keep = _needs_grad(routed, w13, w2)
    return _T.experts(routed, w13, w2, offs, swiglu_limit, keep)[0]


def combine(y, scores_flat, sorted_indices, inverse, top_k, score_after):
    """out[t] = sum_k w(t,k) * y[pos(t,k)], w = score if score after experts else 1."""
    return _T.combine(y, scores_flat, sorted_indices, inverse, top_k, score_after)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """bf16 x * rsqrt(mean(x^2) + eps) * weight over the last dimension
    (models/common/npu_rmsnorm.py:15-37), the norm in front of a block; x bf16
    or fp32 [..., D], differentiable in x and weight."""
    rows = x.reshape(-1, x.shape[-1])
    return _T.rms_norm(rows, weight, eps, _needs_grad(x, weight))[0].view(x.shape)


def residual_norm(
    branch: torch.Tensor,
    residual: torch.Tensor | None = None,
    post_weight: torch.Tensor | None = None,
    gate: torch.Tensor | None = None,
    gate_func: str = "identity",
    residual_scale: float = 1.0,
    pre_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """(u, n): u = residual + residual_scale * act(gate) * rmsnorm(branch) *
    post_weight, n = rmsnorm(u) * pre_weight (None without pre_weight), rows
    [T, D]; differentiable in every tensor.  Operands as ops.residual_norm."""
    keep = _needs_grad(branch, residual, post_weight, gate, pre_weight)
    u, n, _ = _T.residual_norm(branch.to(_BF16), residual, post_weight, gate, gate_func, residual_scale, pre_weight,
                               eps, keep)
    return u, (None if pre_weight is None else n)


class HIPMoeTokenUnpermute:
    """Functional unpermute with backward; same contract as the reference's
    NPUMoeTokenUnpermute (torchtitanturbo/models/common/npu_permute.py:15-53):
    probs=None, top_k=1, empty input passes through.  With one choice per
    row and no probs the unpermute is a pure row scatter,
    out[sorted_indices[j]] = permuted_tokens[j], and its backward the
    matching gather (ttamd::token_unpermute), so both move rows bit for bit
    in the input's dtype."""

    @staticmethod
    def apply(permuted_tokens, sorted_indices, restore_shape):
        if not permuted_tokens.numel():
            return permuted_tokens
        rows = permuted_tokens.reshape(-1, permuted_tokens.shape[-1])
        return _T.token_unpermute(rows, sorted_indices).view(restore_shape)


def token_permute(rows, labels, num_labels):
    """permuted[j] = rows[sorted_indices[j]], sorted_indices the stable order of
    the row labels (torch_npu.npu_moe_token_permute with one label per row,
    npu_permute.py:74-76).  Rows move bit for bit in their own dtype; the
    backward scatters the gradient rows back, grad_rows[sorted_indices[j]] =
    grad_permuted[j] (ttamd::token_permute)."""
    return _T.token_permute(rows, labels, num_labels)


def run_experts_grouped_mm(
    w13: torch.Tensor,
    w2: torch.Tensor,
    x: torch.Tensor,
    num_tokens_per_expert: torch.Tensor,
    swiglu_limit: float | None = None,
) -> torch.Tensor:
    """Same signature and result as the reference's _run_experts_grouped_mm
    (torchtitanturbo/models/common/npu_gmm.py:21-40), on the HIP kernels."""
    offs = torch.cumsum(num_tokens_per_expert, dim=0, dtype=torch.int32)
    y = experts(x.to(_BF16).contiguous(), w13, w2, offs, swiglu_limit)
    return y.type_as(x)


def shared_expert_combine(
    routed_out: torch.Tensor,
    x: torch.Tensor,
    w13_shared: torch.Tensor,
    w2_shared: torch.Tensor,
    gate_logits: torch.Tensor | None = None,
    swiglu_limit: float | None = None,
) -> torch.Tensor:
    """routed_out + g * shared_expert(x), g = sigmoid(gate_logits) or 1
    (torchtitanturbo/models/qwen3_5/model.py:796-809; UPSTREAM Llama4 adds the
    ungated shared expert).  x [T, D]; w13_shared [2H, D]; w2_shared [D, H].

    Without autograd this is one fused pass (ttamd::shared_expert_add: the
    shared w2 GEMM adds into the routed output in its epilogue).  With
    autograd it runs the shared FFN as a one-expert ttamd::experts and
    composes the gate and the sum in torch, so every input gets its
    gradient."""
    if not _needs_grad(routed_out, x, w13_shared, w2_shared, gate_logits):
        return _T.shared_expert_add(routed_out, x, w13_shared, w2_shared, gate_logits, swiglu_limit)
    T = x.shape[0]
    all_rows = torch.full((1,), T, dtype=torch.int32, device=x.device)
    y = experts(x.to(_BF16).contiguous(), w13_shared.unsqueeze(0), w2_shared.unsqueeze(0), all_rows, swiglu_limit)
    if gate_logits is not None:
        y = torch.sigmoid(gate_logits.to(y.dtype)).reshape(T, 1) * y
    return routed_out + y


def _check_checkpoint(checkpoint: str | None) -> None:
    if checkpoint not in (None, "e4m3"):
        raise ValueError(f"checkpoint must be 'e4m3' or None, got {checkpoint!r}")


def moe_experts_forward(
    x: torch.Tensor,
    top_scores: torch.Tensor,
    selected_experts_indices: torch.Tensor,
    w13: torch.Tensor,
    w2: torch.Tensor,
    num_experts: int,
    score_before_experts: bool,
    swiglu_limit: float | None = None,
    stage_events: dict | None = None,
    checkpoint: str | None = None,
) -> torch.Tensor:
    """dispatch -> experts -> combine for one GPU; x [T, D], scores/indices [T, K] -> [T, D].

    ``checkpoint="e4m3"`` keeps the activations that the backward needs in 8
    bits (x, the pre-activation and the experts' outputs, packed by
    ops.pack_e4m3): about a third of the bf16 ones' memory (a quarter with
    many choices per token).  The output is the same; the weights' and the
    scores' gradients are those at the stored values: within 2^-4 of an
    activation of at least 2^-13 of the largest in its row's 128 columns, a
    smaller one within 2^-17 of that largest (so the least become 0).  A step
    takes longer: 8192 tokens to 8 of 128 experts of 1536 x 2048, 2.40 -> 2.59 ms
    and 107 -> 35 KB kept per token; with fp32 weights, whose bf16 copies
    (1.2 GB here) are made again instead of kept, 3.13 -> 3.97 ms.

    With autograd off (or nothing requiring grad) the expert stage is one
    op (ttamd::moe_experts_forward: both grouped GEMMs on one tile table,
    the score multiply and the un-permute in the w2 GEMM epilogue).
    ``stage_events``, when given (inference path only), runs the same kernels
    one op at a time and receives a (start, end) pair of torch.cuda.Event
    per stage, recorded on the current stream around the stage's kernels:
    {"route", "permute", "gemm_w13_swiglu", "gemm_w2_unpermute", "sum_topk"}.
    """
    T, D = x.shape
    K = top_scores.shape[-1]
    _check_checkpoint(checkpoint)
    if w13.shape[0] != num_experts:
        raise ValueError(f"w13 holds {w13.shape[0]} experts, num_experts is {num_experts}")
    training = _needs_grad(x, top_scores, w13, w2)
    ev = stage_events if (stage_events is not None and not training) else None

    def mark(name: str, end: bool) -> None:
        if ev is not None:
            pair = ev.setdefault(name, (torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)))
            pair[1 if end else 0].record()

    scores_flat = top_scores.reshape(-1).float()
    mark("route", False)
    counts, offsets, sorted_idx, inverse, sorted_scores = _T.route(
        selected_experts_indices.reshape(-1), num_experts, scores_flat.detach())
    mark("route", True)
    offs = offsets[1:]
    xb = x.to(_BF16).contiguous()
    if not training and ev is None and D % 128 == 0:
        out = _T.moe_experts_forward(xb, sorted_idx, offsets, sorted_scores, _bf16(w13), _bf16(w2), K,
                                     score_before_experts, swiglu_limit)
        return out.to(x.dtype)
    if not training:
        # op-at-a-time over the same kernels (stage timing; D < 128)
        r = ops.RouteResult(counts, offsets, sorted_idx, inverse, sorted_scores)
        w13b, w2b = _bf16(w13), _bf16(w2)
        if score_before_experts or D < 128:
            mark("permute", False)
            routed = ops.permute_rows(xb, r, K, scores_flat if score_before_experts else None)
            mark("permute", True)
            mark("gemm_w13_swiglu", False)
            a, _ = ops.grouped_mm_swiglu(routed, w13b, offs, swiglu_limit)
            mark("gemm_w13_swiglu", True)
        else:
            # the permute gather happens inside the w13 GEMM's loads
            mark("gemm_w13_swiglu", False)
            a, _ = ops.grouped_mm_swiglu_gather(xb, r.sorted_indices, K, w13b, offs, swiglu_limit)
            mark("gemm_w13_swiglu", True)
        scale = None if score_before_experts else r.sorted_scores
        if K == 1:
            mark("gemm_w2_unpermute", False)
            out = ops.grouped_mm_unpermute(a, w2b, offs, scale, r.sorted_indices, T)
            mark("gemm_w2_unpermute", True)
        else:
            mark("gemm_w2_unpermute", False)
            ybuf = ops.grouped_mm_unpermute(a, w2b, offs, scale, r.sorted_indices, T * K)
            mark("gemm_w2_unpermute", True)
            mark("sum_topk", False)
            out = ops.sum_topk(ybuf, K)
            mark("sum_topk", True)
        return out.to(x.dtype)
    if checkpoint is not None:
        keep_y = not score_before_experts and scores_flat.requires_grad
        out = _T.experts_packed(xb, scores_flat, sorted_idx, inverse, sorted_scores, offs, w13, w2, K,
                                score_before_experts, swiglu_limit, keep_y)[0]
        return out.to(x.dtype)
    routed = dispatch(xb, scores_flat, sorted_idx, inverse, sorted_scores, K, score_before_experts)
    y = experts(routed, w13, w2, offs, swiglu_limit)
    out = combine(y, scores_flat, sorted_idx, inverse, K, not score_before_experts)
    return out.to(x.dtype)


def _tensors(w) -> tuple:
    """(weights or codes, exponents or None) of weights in either form, or of None."""
    return (w.codes, w.exponents) if isinstance(w, PackedWeights) else (w, None)


def _bf16_weights(w):
    """bf16 [E, N, K] of weights in either form; [N, K] is one expert."""
    w = unpack_e2m1(w) if isinstance(w, PackedWeights) else w
    return w if w.dim() == 3 else w.unsqueeze(0)


def _hidden(w13) -> int:
    return 0 if w13 is None else (w13.rows if isinstance(w13, PackedWeights) else w13.shape[-2]) // 2


_transforms = torch._C._functorch.peek_interpreter_stack
_PLAIN = {torch.Tensor, torch.nn.Parameter, type(None)}


def _as_op(*args) -> bool:
    """Whether something sees the call before the device does (torch.compile, a tracer,
    a dispatch mode, a function transform, a tensor subclass): it takes the registered
    op then.  Else the C call at once: an op's dispatch costs a call on one token more
    than its kernels take."""
    if torch.compiler.is_compiling() or decode._seen() or _transforms() is not None:
        return True
    for t in args:
        if type(t) not in _PLAIN and not (
                type(t) is PackedWeights and type(t.codes) is type(t.exponents) is torch.Tensor):
            return True
    return False


def pack_e2m1(w: torch.Tensor) -> PackedWeights:
    """decode.pack_e2m1, or ttamd::pack_e2m1 under a tracer."""
    if not _as_op(w):
        return decode.pack_e2m1(w)
    decode._no_grad("pack_e2m1", w)
    return PackedWeights(*_T.pack_e2m1(w), *w.shape[-2:])


def unpack_e2m1(w: PackedWeights) -> torch.Tensor:
    """decode.unpack_e2m1, or ttamd::unpack_e2m1 under a tracer."""
    return _T.unpack_e2m1(*w) if _as_op(w) else decode.unpack_e2m1(w)


def grouped_mm_e2m1(
    x: torch.Tensor, w: PackedWeights, offs: torch.Tensor | None = None, bias: torch.Tensor | None = None
) -> torch.Tensor:
    """decode.grouped_mm_e2m1, or ttamd::grouped_mm_e2m1 under a tracer."""
    if not _as_op(x, w, offs, bias):
        return decode.grouped_mm_e2m1(x, w, offs, bias)
    decode._no_grad("grouped_mm_e2m1", x, bias)
    return _T.grouped_mm_e2m1(x, w.codes, w.exponents, w.rows, offs, bias)


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
    """decode.router_decode, or ttamd::router_decode under a tracer."""
    args = (x, w_router, top_k, score_func, route_norm, route_scale, expert_bias, norm_eps, num_groups, topk_groups,
            group_score, shared_gate)
    if not _as_op(x, w_router, expert_bias, shared_gate):
        return decode.router_decode(*args)
    decode._no_grad("router_decode", x, w_router, shared_gate)
    scores, idx, gate = _T.router_decode(*args)
    return scores, idx, None if shared_gate is None else gate


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
    """decode.experts_decode, or ttamd::experts_decode under a tracer."""
    if not _as_op(x, top_scores, selected_experts_indices, w13, w2, shared_w13, shared_w2, shared_scale):
        return decode.experts_decode(x, top_scores, selected_experts_indices, w13, w2, score_before_experts,
                                     swiglu_limit, shared_w13, shared_w2, shared_scale)
    decode._no_grad("experts_decode", x, top_scores, w13, w2, shared_w13, shared_w2, shared_scale)
    (t13, e13), (t2, e2), (u13, f13), (u2, f2) = map(_tensors, (w13, w2, shared_w13, shared_w2))
    return _T.experts_decode(x, top_scores, selected_experts_indices, t13, t2, _hidden(w13), score_before_experts,
                             swiglu_limit, e13, e2, _hidden(shared_w13), u13, u2, f13, f2, shared_scale)


def _prompt_router(x, w_router, top_k, func, norm, scale, bias, eps, num_groups, topk_groups, group_score):
    """functional.router for as many experts as the few-token layer takes: the fused gate
    holds 256, so of more the logits come from it run by run, and the selection from them
    (with groups, whose 64-bit form that layer's selection is)."""
    if w_router.shape[0] <= 256:
        return router(x, w_router, top_k, func, norm, scale, bias, eps, num_groups, topk_groups, group_score)
    x = x.contiguous()
    logits = torch.cat([_T.router(x, w, 1, func, False, 1.0, None, eps)[2] for w in w_router.split(256)], 1)
    if num_groups is None and topk_groups is None:
        num_groups = topk_groups = 1
    return router_topk(logits, top_k, func, norm, scale, bias, eps, num_groups, topk_groups, group_score)


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
    """The MoE layer of a serving step on one GPU, for batches of any length: x bf16
    [T, D] to (out bf16 [T, D], top_scores fp32 [T, K], selected_experts_indices
    int64 [T, K]); arguments as decode.moe_decode.  At most 64 tokens stream the
    weights (decode.moe_decode; under a tracer ttamd::moe_decode); a prompt takes
    the router, the grouped GEMMs and the shared expert's pass, 4-bit weights
    restored to bf16 for the call (D % 128 == 0 and H % 64 == 0 there, a shared
    expert's H too).  The two sum a logit in other orders, so tokens whose experts
    nearly tie may pick others.  No backward."""
    decode._no_grad("moe_decode", x, w_router, w13, w2, shared_w13, shared_w2, shared_gate)
    if x.dim() != 2 or x.dtype != _BF16:
        raise TypeError(f"x must be bfloat16 [T, D], got {x.dtype} {tuple(x.shape)}")
    if x.shape[0] > decode.MAX_TOKENS:
        if (shared_w13 is None) != (shared_w2 is None):
            raise ValueError("give shared_w13 and shared_w2 together")
        if shared_gate is not None and shared_w13 is None:
            raise ValueError("shared_gate needs a shared expert")
        for name, w in (("w_router", w_router), ("w13", w13), ("w2", w2), ("shared_w13", shared_w13),
                        ("shared_w2", shared_w2), ("shared_gate", shared_gate), ("expert_bias", expert_bias)):
            packed = isinstance(w, PackedWeights)
            if w is not None and not packed and w.dtype != _BF16 and w is not expert_bias:
                raise TypeError(f"{name} must be bfloat16, got {w.dtype}")
            for t in w[:2] if packed else (w,):
                if t is not None and t.device != x.device:  # (a kernel would read through its pointer)
                    raise RuntimeError(f"{name} is on {t.device}, expected {x.device}")
        if isinstance(w13, PackedWeights) != isinstance(w2, PackedWeights):
            raise TypeError("w13 and w2 must both be bfloat16 or both packed")
        if any(w is not None and isinstance(w, PackedWeights) != isinstance(w13, PackedWeights)
               for w in (shared_w13, shared_w2)):
            raise TypeError("the shared expert's weights must be of the experts' type")
        scores, idx = _prompt_router(x, w_router, top_k, score_func, route_norm, route_scale, expert_bias, norm_eps,
                                     num_groups, topk_groups, group_score)
        out = moe_experts_forward(x, scores, idx, _bf16_weights(w13), _bf16_weights(w2), w_router.shape[0],
                                  score_before_experts, swiglu_limit)
        if shared_w13 is not None:
            s13, s2 = (w.reshape(w.shape[-2:]) for w in map(_bf16_weights, (shared_w13, shared_w2)))
            logits = None if shared_gate is None else x @ shared_gate.reshape(-1)
            out = shared_expert_combine(out, x, s13, s2, logits, swiglu_limit)
        return out, scores, idx
    if not _as_op(x, w_router, w13, w2, expert_bias, shared_w13, shared_w2, shared_gate):
        return decode.moe_decode(x, w_router, w13, w2, top_k, score_func, route_norm, route_scale, expert_bias,
                                 norm_eps, num_groups, topk_groups, group_score, score_before_experts, swiglu_limit,
                                 shared_w13, shared_w2, shared_gate)
    (t13, e13), (t2, e2), (u13, f13), (u2, f2) = map(_tensors, (w13, w2, shared_w13, shared_w2))
    return _T.moe_decode(x, w_router, t13, t2, top_k, _hidden(w13), score_func, route_norm, route_scale, expert_bias,
                         norm_eps, num_groups, topk_groups, group_score, score_before_experts, swiglu_limit, e13, e2,
                         _hidden(shared_w13), u13, u2, f13, f2, shared_gate)


def moe_block(
    x: torch.Tensor,
    w_router: torch.Tensor,
    w13: torch.Tensor,
    w2: torch.Tensor,
    top_k: int,
    pre_weight: torch.Tensor | None = None,
    post_weight: torch.Tensor | None = None,
    gate: torch.Tensor | None = None,
    gate_func: str = "identity",
    residual_scale: float = 1.0,
    next_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    score_func: str = "softmax",
    route_norm: bool = False,
    route_scale: float = 1.0,
    expert_bias: torch.Tensor | None = None,
    num_groups: int | None = None,
    topk_groups: int | None = None,
    group_score: str = "top2",
    score_before_experts: bool = False,
    swiglu_limit: float | None = None,
    checkpoint: str | None = None,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """One MoE block of a transformer on one GPU: x [T, D] (the residual stream,
    bf16 or fp32) to (u, n),

        h = rmsnorm(x) * pre_weight             (None: x itself)
        f = experts of h's routing, combined    (router, moe_experts_forward)
        u = x + residual_scale * act(gate) * rmsnorm(f) * post_weight
        n = rmsnorm(u) * next_weight            (None without next_weight)

    in the places of upstream's TransformerBlock ffn_norm, moe and residual sum
    and the next block's first norm.  With autograd every piece carries its
    registered backward; without, the norms after the block run inside the
    combine (ops.combine_norm).  Routing arguments as `router`, checkpoint as
    `moe_experts_forward`, norm arguments as `residual_norm`; D % 128 == 0."""
    _check_checkpoint(checkpoint)
    if w_router.shape[0] != w13.shape[0]:
        raise ValueError(f"w_router chooses among {w_router.shape[0]} experts, w13 holds {w13.shape[0]}")
    groups = dict(num_groups=num_groups, topk_groups=topk_groups, group_score=group_score)
    how = dict(post_weight=post_weight, gate=gate, gate_func=gate_func, residual_scale=residual_scale,
               pre_weight=next_weight, eps=eps)
    if not _needs_grad(x, w_router, w13, w2, pre_weight, post_weight, gate, next_weight):
        u, n = _T.moe_block_forward(x, w_router, w13, w2, top_k, pre_weight, post_weight, gate, gate_func,
                                    residual_scale, next_weight, eps, score_func, route_norm, route_scale,
                                    expert_bias, num_groups, topk_groups, group_score, score_before_experts,
                                    swiglu_limit)
        return u, (None if next_weight is None else n)
    h = x.to(_BF16) if pre_weight is None else rms_norm(x, pre_weight, eps)
    scores, idx = router(h, w_router, top_k, score_func, route_norm, route_scale, expert_bias, **groups)
    f = moe_experts_forward(h, scores, idx, w13, w2, w13.shape[0], score_before_experts, swiglu_limit,
                            checkpoint=checkpoint)
    return residual_norm(f, x, **how)


def moe_experts_forward_fp8(
    x: torch.Tensor,
    top_scores: torch.Tensor,
    selected_experts_indices: torch.Tensor,
    w13q: torch.Tensor,
    s13: torch.Tensor,
    w2q: torch.Tensor,
    s2: torch.Tensor,
    num_experts: int,
    score_before_experts: bool,
    swiglu_limit: float | None = None,
    stage_events: dict | None = None,
) -> torch.Tensor:
    """Inference forward with fp8 e4m3 experts (weights pre-quantised with
    ops.quantize_fp8_blocks): route -> gather + per-token quantise -> fp8
    w13 + SwiGLU -> per-token re-quantise of a -> fp8 w2 + scale + scatter
    -> K-way sum.  x [T, D] bf16 -> [T, D]."""
    T, D = x.shape
    K = top_scores.shape[-1]
    ev = stage_events

    def mark(name: str, end: bool) -> None:
        if ev is not None:
            pair = ev.setdefault(name, (torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)))
            pair[1 if end else 0].record()

    scores_flat = top_scores.reshape(-1).float()
    mark("route", False)
    r = ops.route(selected_experts_indices, num_experts, scores_flat)
    mark("route", True)
    xb = x.to(_BF16).contiguous()
    mark("permute_quantize", False)
    xq, sx = ops.quantize_fp8_rows(xb, r.sorted_indices, K, r.sorted_scores if score_before_experts else None)
    mark("permute_quantize", True)
    mark("gemm_w13_swiglu", False)
    a, _ = ops.grouped_mm_fp8_swiglu(xq, sx, w13q, s13, r.offs, swiglu_limit)
    mark("gemm_w13_swiglu", True)
    mark("quantize_a", False)
    aq, sa = ops.quantize_fp8_rows(a)
    mark("quantize_a", True)
    scale = None if score_before_experts else r.sorted_scores
    mark("gemm_w2_unpermute", False)
    if K == 1:
        out = ops.grouped_mm_fp8_unpermute(aq, sa, w2q, s2, r.offs, scale, r.sorted_indices, T)
        mark("gemm_w2_unpermute", True)
    else:
        ybuf = ops.grouped_mm_fp8_unpermute(aq, sa, w2q, s2, r.offs, scale, r.sorted_indices, T * K)
        mark("gemm_w2_unpermute", True)
        mark("sum_topk", False)
        out = ops.sum_topk(ybuf, K)
        mark("sum_topk", True)
    return out.to(x.dtype)
