"""Measured operators around and inside the MoE block: group-limited routing,
the norms before and after the block with its gate and residual scale, the
combine that ends in them, and 8-bit activation checkpoints with the backward
products that read them.

A case is a dict of plain values; ``kind`` names the operator:

  route      top-k routing limited to groups of experts, from given logits;
             with ``train`` also the gradient of the logits
  norm       p = rmsnorm(f) * w_post; u = residual + scale * act(gate) * p;
             n = rmsnorm(u) * w_pre; with ``train`` also every gradient
  combine    the same with f the score-weighted sum of a token's expert rows
  store      rows packed to 8 bits and restored: what a checkpoint gives back
  dgrad      d(pre-activation) and the activation of the expert FFN from the
             packed pre-activation and dy . w2
  wgrad      the expert weight gradient dy^T . x from packed token rows,
             gathered in routing order

``own`` chooses between the plain form (torch operations in 32 bits, 64 where
selections or values next to a border need them) and the framework's calls.
"""
from __future__ import annotations

import importlib
import math

import torch

own = False

_PKG = "torchtitan-ascend_amd"
_DEV = "cuda"
_BF16 = torch.bfloat16
_EPS = 1e-6
_NORM_EPS = 1e-20
_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _route(T, E, K, groups, kept, func, value, **o):
    return dict(dict(kind="route", T=T, E=E, K=K, groups=groups, kept=kept, func=func, value=value, bias=True,
                     renorm=True, scale=2.5, logits="fp32", train=False), **o)


def _norm(T, D, **o):
    return dict(dict(kind="norm", T=T, D=D, post=True, pre=True, residual=True, gate="none", act="identity",
                     scale=1.0, stream="bf16", weights="bf16", train=False), **o)


def _combine(T, D, K, **o):
    return dict(dict(_norm(T, D), kind="combine", K=K, gathered=True, scored=True), **o)


def _experts(kind, T, K, E, D, H, **o):
    return dict(dict(kind=kind, T=T, K=K, E=E, D=D, H=H, skew=0.3, empty=0, limit=0.0), **o)


def listed():
    cases = [
        # a decode batch of a model with 256 experts in 8 groups, 4 of them kept
        ("route_decode_32", _route(32, 256, 8, 8, 4, "sigmoid", "top2")),
        # a full prefill batch of the same model
        ("route_prefill_16384", _route(16384, 256, 8, 8, 4, "sigmoid", "top2")),
        # a ragged training micro-batch with softmax scores and groups by their best expert
        ("route_train_4099", _route(4099, 160, 6, 8, 3, "softmax", "max", bias=False, renorm=False, logits="bf16",
                                    train=True)),
        # one sequence decoding: the end of one block and the norm of the next
        ("norm_decode_1", _norm(1, 7168, gate="token", act="sigmoid")),
        # a training step of a 5120-wide block, per-channel gate, fp32 weights
        ("norm_train_8192x5120", _norm(8192, 5120, gate="channel", scale=0.5, weights="fp32", train=True)),
        # a small odd-sized training step with an fp32 residual stream and an element-wise gate
        ("norm_train_1003x2056", _norm(1003, 2056, gate="full", act="sigmoid", stream="fp32", train=True)),
        # a decode batch: eight expert rows per token in token order
        ("combine_decode_64", _combine(64, 2048, 8, gathered=False, scored=False)),
        # a full prefill batch: eight rows per token, gathered from expert order and weighted
        ("combine_prefill_8192", _combine(8192, 2048, 8, gate="token", act="sigmoid")),
        # a short ragged micro-batch's pre-activation stored and restored
        ("store_1003x1544", dict(kind="store", R=1003, C=1544)),
        # the pre-activation of a full micro-batch over 128 experts (2 H = 1536)
        ("store_65536x1536", dict(kind="store", R=65536, C=1536)),
        # an expert shard's backward through the activation: 32 experts, uneven load
        ("dgrad_32x7168x2048", _experts("dgrad", 32768, 1, 32, 7168, 2048, skew=0.7, empty=2)),
        # the weight gradient of 128 small experts, top-8 rows gathered from packed tokens
        ("wgrad_128x1536x2048", _experts("wgrad", 8192, 8, 128, 2048, 768)),
    ]
    return [dict(c, name=n) for n, c in cases]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    kind = rng.choice(["route", "route", "norm", "norm", "combine", "store", "dgrad", "wgrad"])
    if kind == "route":
        E = rng.choice([16, 60, 64, 128, 160, 256])
        groups = rng.choice([g for g in (1, 2, 4, 5, 8, 10, 16) if E % g == 0])
        kept = rng.randint(1, groups)
        K = rng.randint(1, min(16, kept * (E // groups)))
        return _route(_log_int(rng, 1, 16384), E, K, groups, kept, rng.choice(["sigmoid", "softmax"]),
                      rng.choice(["top2", "max"]), bias=rng.random() < 0.6,
                      renorm=K > 1 and rng.random() < 0.6,  # a single renormalised weight is 1, without a gradient
                      scale=rng.choice([1.0, 2.5]), logits=rng.choice(["fp32", "bf16"]), train=rng.random() < 0.4)
    if kind in ("norm", "combine"):
        o = dict(gate=rng.choice(["none", "token", "channel", "full"]), act=rng.choice(["identity", "sigmoid"]),
                 post=rng.random() < 0.8, pre=rng.random() < 0.8, residual=rng.random() < 0.85,
                 scale=rng.choice([1.0, 0.22]), stream=rng.choice(["bf16", "bf16", "fp32"]),
                 weights=rng.choice(["bf16", "fp32"]))
        D = 8 * _log_int(rng, 8, 640 if kind == "norm" else 256)
        T = _log_int(rng, 1, 8192)
        if kind == "norm":
            return _norm(T, D, train=rng.random() < 0.6, **o)
        K = rng.choice([1, 2, 4, 6, 8])
        return _combine(T, D, K, gathered=rng.random() < 0.6, scored=rng.random() < 0.6, **o)
    if kind == "store":
        return dict(kind="store", R=_log_int(rng, 1, 65536), C=8 * _log_int(rng, 4, 192))
    D, H = 128 * rng.randint(2, 16), 128 * rng.randint(1, 8)
    E = rng.choice([1, 4, 16, 64])
    return _experts(kind, _log_int(rng, 4, 4096), rng.choice([1, 2, 8]), E, D, H, skew=rng.choice([0.0, 0.3, 0.7]),
                    empty=rng.choice([0, E // 4]), limit=rng.choice([0.0, 0.0, 1.0]))


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _counts(case):
    """Rows per expert: a power law over the experts that get any."""
    E, rows = case["E"], case["T"] * case["K"]
    n = E - case["empty"]
    w = [(i + 1) ** -case["skew"] for i in range(n)]
    c = [int(rows * x / sum(w)) for x in w]
    c[0] += rows - sum(c)
    order = torch.randperm(E, generator=torch.Generator().manual_seed(E)).tolist()
    at = dict(zip(order, c))
    return [at.get(e, 0) for e in range(E)]


def _pack_plain(x):
    """(codes [R, C] e4m3 bits, exponent bytes [R, ceil(C / 128)]) of bf16 rows: per row and 128 columns the
    smallest power of two 2^e with max|v| <= 448 * 2^e, stored as e + 127."""
    R, C = x.shape
    nb = (C + 127) // 128
    v = torch.nn.functional.pad(x.float(), (0, nb * 128 - C)).view(R, nb, 128)
    m, e = torch.frexp(v.abs().amax(2))  # absmax = m 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = (e - 9 + (m > 0.875).int()).clamp(-118, 120)
    e = torch.where(m == 0, torch.full_like(e, -118), e)
    codes = torch.ldexp(v, -e.unsqueeze(2)).to(torch.float8_e4m3fn).view(torch.uint8)
    return codes.view(R, nb * 128)[:, :C].contiguous(), (e + 127).to(torch.uint8)


def prepare(case, seed):
    gen = torch.Generator(device=_DEV)
    gen.manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0, dtype=_BF16):
        return (torch.randn(*shape, generator=gen, device=_DEV) * std + mean).to(dtype)

    kind = case["kind"]
    s = dict(case=case)
    if kind == "route":
        T, E = case["T"], case["E"]
        s["logits"] = normal(T, E, std=1.5, dtype=_TYPES[case["logits"]])
        s["bias"] = normal(E, std=0.05, dtype=torch.float32) if case["bias"] else None
        s["grad"] = normal(T, case["K"], dtype=torch.float32) if case["train"] else None
    elif kind in ("norm", "combine"):
        T, D = case["T"], case["D"]
        wt, st = _TYPES[case["weights"]], _TYPES[case["stream"]]
        if kind == "combine":
            M = T * case["K"]
            s["rows"] = normal(M, D)
            s["inverse"] = torch.randperm(M, generator=gen, device=_DEV).int() if case["gathered"] else None
            s["probs"] = torch.rand(T, case["K"], generator=gen, device=_DEV) if case["scored"] else None
        else:
            s["branch"] = normal(T, D)
        s["residual"] = normal(T, D, std=3.0, dtype=st) if case["residual"] else None
        s["post"] = normal(D, std=0.2, mean=1.0, dtype=wt) if case["post"] else None
        s["pre"] = normal(D, std=0.2, mean=1.0, dtype=wt) if case["pre"] else None
        shape = {"none": None, "token": (T, 1), "channel": (1, D), "full": (T, D)}[case["gate"]]
        s["gate"] = None if shape is None else normal(*shape, dtype=torch.float32 if shape[1] == 1 else wt)
        if case["train"]:
            s["du"] = normal(T, D, dtype=st if case["residual"] else _BF16)
            s["dn"] = normal(T, D) if case["pre"] else None
    elif kind == "store":
        # activations: most values small, some columns large
        s["x"] = (normal(case["R"], case["C"]).float() * torch.exp2(normal(1, case["C"], std=2.0).float())).to(_BF16)
    else:
        T, K, E, D, H = (case[k] for k in ("T", "K", "E", "D", "H"))
        M = T * K
        counts = _counts(case)
        s["offs"] = torch.tensor(counts, device=_DEV).cumsum(0).int()
        s["cap"] = max(counts)
        if kind == "dgrad":
            s["dy"] = normal(M, D)
            s["w2"] = normal(E, D, H, std=0.02)
            s["h"] = _pack_plain(normal(M, 2 * H))
        else:
            s["dy"] = normal(M, 2 * H)
            s["x"] = _pack_plain(normal(T, D))
            s["src"] = torch.randperm(M, generator=gen, device=_DEV).int()
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    ops = importlib.import_module(_PKG + ".ops")
    c = s["case"]
    kind = c["kind"]
    if kind == "route":
        scores, idx = ops.router_topk(s["logits"], c["K"], c["func"], c["renorm"], c["scale"], s["bias"], _NORM_EPS,
                                      num_groups=c["groups"], topk_groups=c["kept"], group_score=c["value"])
        if not c["train"]:
            return scores, idx
        return scores, idx, ops.router_topk_backward(s["grad"], idx, s["logits"], c["func"], c["renorm"], c["scale"],
                                                     _NORM_EPS)
    if kind in ("norm", "combine"):
        how = dict(residual=s["residual"], post_weight=s["post"], gate=s["gate"], gate_func=c["act"],
                   residual_scale=c["scale"], pre_weight=s["pre"], eps=_EPS)
        if kind == "combine":
            return ops.combine_norm(s["rows"], c["K"], inverse=s["inverse"], probs=s["probs"], **how)
        if not c["train"]:
            return ops.residual_norm(s["branch"], **how)
        u, n, stats = ops.residual_norm(s["branch"], save_stats=True, **how)
        return u, n, tuple(ops.residual_norm_backward(s["du"], s["dn"], s["branch"], stats, **how))
    if kind == "store":
        return ops.unpack_e4m3(ops.pack_e4m3(s["x"]))
    if kind == "dgrad":
        return ops.grouped_mm_dgrad_swiglu_packed(s["dy"], s["w2"], ops.PackedRows(*s["h"]), s["offs"],
                                                  c["limit"] or None, want_a=True)
    return ops.grouped_mm_wgrad_packed(s["dy"], ops.PackedRows(*s["x"]), s["offs"], c["E"], src_index=s["src"],
                                       src_div=c["K"])


def _plain(s):
    return {"route": _plain_route, "norm": _plain_norm, "combine": _plain_norm, "store": _plain_store,
            "dgrad": _plain_dgrad, "wgrad": _plain_wgrad}[s["case"]["kind"]](s)


def _plain_route(s):
    """Scores and selection in 64 bits: two candidates closer than a 32-bit ulp are common."""
    c = s["case"]
    T, E, G, K = c["T"], c["E"], c["groups"], c["K"]
    z = s["logits"].double()
    if c["func"] == "softmax":
        ex = torch.exp(z - z.amax(1, keepdim=True))
        p = ex / ex.sum(1, keepdim=True)
    else:
        p = 1.0 / (1.0 + torch.exp(-z))
    v = p if s["bias"] is None else p + s["bias"].double()
    top = torch.sort(v.view(T, G, E // G), dim=2, descending=True).values
    value = top[:, :, :2].sum(2) if c["value"] == "top2" else top[:, :, 0]
    kept = torch.sort(value, dim=1, descending=True, stable=True).indices[:, :c["kept"]]
    mask = torch.zeros(T, G, dtype=torch.bool, device=z.device).scatter_(1, kept, True)
    v = v.masked_fill(~mask.repeat_interleave(E // G, 1), -math.inf)
    idx = torch.sort(v, dim=1, descending=True, stable=True).indices[:, :K].contiguous()
    w = p.gather(1, idx)
    total = w.sum(1, keepdim=True) + _NORM_EPS
    scores = ((w / total if c["renorm"] else w) * c["scale"]).float()
    if not c["train"]:
        return scores, idx
    g = s["grad"].double() * c["scale"]
    if c["renorm"]:
        g = g / total - (g * w).sum(1, keepdim=True) / (total * total)
    dp = torch.zeros_like(p).scatter_(1, idx, g)
    if c["func"] == "softmax":
        dz = p * (dp - (dp * p).sum(1, keepdim=True))
    else:
        dz = dp * p * (1.0 - p)
    return scores, idx, dz.to(s["logits"].dtype)


def _combined(s):
    c = s["case"]
    rows = s["rows"].float()
    if s["inverse"] is not None:
        rows = rows[s["inverse"].long()]
    rows = rows.view(c["T"], c["K"], c["D"])
    if s["probs"] is not None:
        rows = rows * s["probs"].unsqueeze(2)
    return rows.sum(1)


def _plain_norm(s):
    c = s["case"]
    f = _combined(s) if c["kind"] == "combine" else s["branch"].float()
    out_type = s["residual"].dtype if s["residual"] is not None else _BF16
    r_f = torch.rsqrt((f * f).mean(1, keepdim=True) + _EPS)
    f_hat = f * r_f
    p = f_hat * s["post"].float() if c["post"] else f
    raw = None if s["gate"] is None else s["gate"].float()
    a = 1.0 if raw is None else (1.0 / (1.0 + torch.exp(-raw)) if c["act"] == "sigmoid" else raw)
    u = c["scale"] * a * p
    if s["residual"] is not None:
        u = u + s["residual"].float()
    r_u = torch.rsqrt((u * u).mean(1, keepdim=True) + _EPS)
    n = (u * r_u * s["pre"].float()).to(_BF16) if c["pre"] else None
    if not c["train"]:
        return u.to(out_type), n
    d_u, d_pre = s["du"].float(), None
    if c["pre"]:
        dn, u_hat = s["dn"].float(), u * r_u
        q = dn * s["pre"].float()
        d_pre = (dn * u_hat).sum(0).to(s["pre"].dtype)
        d_u = d_u + r_u * (q - u_hat * (q * u_hat).mean(1, keepdim=True))
    d_res = d_u.to(out_type) if s["residual"] is not None else None
    d_gate = None
    if raw is not None:
        da = c["scale"] * d_u * p
        if c["act"] == "sigmoid":
            da = da * a * (1.0 - a)
        if raw.shape[1] == 1 and c["D"] > 1:
            da = da.sum(1, keepdim=True)
        elif c["gate"] == "channel":
            da = da.sum(0, keepdim=True)
        d_gate = da.to(s["gate"].dtype)
    d_p = c["scale"] * a * d_u
    d_post = None
    if c["post"]:
        d_post = (d_p * f_hat).sum(0).to(s["post"].dtype)
        q = d_p * s["post"].float()
        d_f = r_f * (q - f_hat * (q * f_hat).mean(1, keepdim=True))
    else:
        d_f = d_p
    return u.to(out_type), n, (d_f.to(_BF16), d_res, d_post, d_gate, d_pre)


def _unpack_plain(codes, exps):
    """fp32 values of packed rows."""
    R, C = codes.shape
    e = (exps.int() - 127).repeat_interleave(128, 1)[:, :C]
    return torch.ldexp(codes.view(torch.float8_e4m3fn).float(), e)


def _plain_store(s):
    return _unpack_plain(*_pack_plain(s["x"])).to(_BF16)


def _segments(s, M):
    """Row of place (expert, position) in a table of `cap` places per expert, whether it is one, and each row's expert."""
    offs = s["offs"].long()
    start = torch.cat([offs.new_zeros(1), offs[:-1]])
    row = start.unsqueeze(1) + torch.arange(s["cap"], device=offs.device)
    held = row < offs.unsqueeze(1)
    at = torch.arange(M, device=offs.device)
    expert = torch.searchsorted(offs, at, right=True)
    return row.clamp(max=M - 1), held.unsqueeze(2), expert, at - start[expert]


def _plain_dgrad(s):
    c = s["case"]
    H, limit = c["H"], c["limit"]
    row, held, expert, place = _segments(s, s["dy"].shape[0])
    g = torch.bmm(s["dy"].float()[row] * held, s["w2"].float())[expert, place]
    h = _unpack_plain(*s["h"])
    gate, up = h[:, :H], h[:, H:]
    gc, uc = (gate.clamp(max=limit), up.clamp(-limit, limit)) if limit else (gate, up)
    sig = 1.0 / (1.0 + torch.exp(-gc))
    silu = gc * sig
    dgate, dup = g * uc * (sig * (1.0 + gc * (1.0 - sig))), g * silu
    if limit:
        dgate, dup = dgate * (gate <= limit), dup * (up.abs() <= limit)
    return torch.cat([dgate, dup], 1).to(_BF16), (silu * uc).to(_BF16)


def _plain_wgrad(s):
    c = s["case"]
    row, held, _, _ = _segments(s, s["dy"].shape[0])
    x = _unpack_plain(*s["x"])[s["src"].long() // c["K"]]
    dy = (s["dy"].float()[row] * held).transpose(1, 2).contiguous()
    return torch.bmm(dy, x[row])


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "route":
        T, E, K = case["T"], case["E"], case["K"]
        size = 4 if case["logits"] == "fp32" else 2
        b = T * E * size + 12 * T * K + 4 * E * case["bias"]
        if case["train"]:
            b += T * E * size + 4 * T * K
        return {"bytes": b, "flops": 0}
    if kind in ("norm", "combine"):
        T, D, st = case["T"], case["D"], 4 if case["stream"] == "fp32" else 2
        out = st if case["residual"] else 2
        ws = 4 if case["weights"] == "fp32" else 2
        gate = {"none": 0, "token": 4 * T, "channel": D * ws, "full": T * D * ws}[case["gate"]]
        weights = D * ws * (case["post"] + case["pre"])
        b = T * D * ((st if case["residual"] else 0) + out + 2 * case["pre"]) + gate + weights
        if kind == "combine":
            b += 2 * T * case["K"] * D + 4 * T * case["K"] * (case["gathered"] + case["scored"])
        else:
            b += 2 * T * D
        if case["train"]:
            # the upstream gradients in, the gradients out
            b += T * D * (out + 2 * case["pre"] + 2 + (st if case["residual"] else 0)) + gate + weights
        return {"bytes": b, "flops": 0}
    if kind == "store":
        return {"bytes": 4 * case["R"] * case["C"], "flops": 0}
    T, K, E, D, H = (case[k] for k in ("T", "K", "E", "D", "H"))
    M, hit = T * K, sum(n > 0 for n in _counts(case))
    if kind == "dgrad":
        b = 2 * M * D + 2 * hit * D * H + 2 * M * H * (1 + 1 / 128) + 6 * M * H + 4 * E
        return {"bytes": b, "flops": 2 * M * D * H}
    return {"bytes": 4 * M * H + T * D * (1 + 1 / 128) + 4 * M + 4 * E + 8 * E * H * D, "flops": 4 * M * D * H}


# ---------------------------------------------------------------------------
# The definitions in 64 bits; gradients by torch's autograd
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "route":
        return _exact_route(s)
    if kind in ("norm", "combine"):
        return _exact_norm(s)
    if kind == "store":
        return _exact_store(s)
    return _exact_experts(s)


def _exact_route(s):
    c = s["case"]
    _, idx, *_ = _plain_route(s)  # the selection; the values below are computed apart
    z = s["logits"].double().requires_grad_(c["train"])
    p = torch.softmax(z, 1) if c["func"] == "softmax" else torch.sigmoid(z)
    w = torch.gather(p, 1, idx)
    if c["renorm"]:
        w = w / (w.sum(1, keepdim=True) + _NORM_EPS)
    w = w * c["scale"]
    if not c["train"]:
        return w, None
    (dz,) = torch.autograd.grad(w, z, s["grad"].double())
    return w.detach(), None, dz


def _exact_norm(s):
    c = s["case"]
    wide = {k: s[k].double().requires_grad_(c["train"]) for k in ("branch", "residual", "post", "gate", "pre")
            if s.get(k) is not None}
    if c["kind"] == "combine":
        order = torch.arange(c["T"] * c["K"], device=_DEV) if s["inverse"] is None else s["inverse"].long()
        probs = torch.ones(c["T"], c["K"], device=_DEV) if s["probs"] is None else s["probs"]
        f = (s["rows"][order].double() * probs.double().view(-1, 1)).unflatten(0, (c["T"], c["K"])).sum(1)
    else:
        f = wide["branch"]
    p = f
    if "post" in wide:
        p = f / torch.sqrt(f.square().mean(1, keepdim=True) + _EPS) * wide["post"]
    if "gate" in wide:
        p = p * (torch.sigmoid(wide["gate"]) if c["act"] == "sigmoid" else wide["gate"])
    u = p * c["scale"]
    if "residual" in wide:
        u = u + wide["residual"]
    n = u / torch.sqrt(u.square().mean(1, keepdim=True) + _EPS) * wide["pre"] if "pre" in wide else None
    if not c["train"]:
        return u, n
    outs, grads = ([u], [s["du"].double()]) if n is None else ([u, n], [s["du"].double(), s["dn"].double()])
    got = dict(zip(wide, torch.autograd.grad(outs, list(wide.values()), grads)))
    return (u.detach(), None if n is None else n.detach(),
            tuple(got.get(k) for k in ("branch", "residual", "post", "gate", "pre")))


def _exact_store(s):
    """Each value rounded, ties to even, to the grid of 3 binary places below its own power of two (at least 2^-6)
    after the division by its block's power of two, which is found as a logarithm."""
    x = s["x"].double()
    R, C = x.shape
    block = torch.arange(C, device=x.device) // 128
    most = torch.zeros(R, (C + 127) // 128, dtype=torch.float64, device=x.device)
    most = most.scatter_reduce(1, block.expand(R, C), x.abs(), "amax")
    scale = torch.exp2(torch.ceil(torch.log2(most / 448.0)).clamp(-118, 120))[:, block]
    v = x / scale
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step * scale


def _values64(codes, exps):
    R, C = codes.shape
    scale = torch.exp2(exps.double() - 127.0)
    return codes.view(torch.float8_e4m3fn).double() * scale[:, torch.arange(C, device=codes.device) // 128]


def _exact_experts(s):
    c = s["case"]
    ends = s["offs"].tolist()
    spans = list(zip([0] + ends[:-1], ends))
    if c["kind"] == "wgrad":
        x = _values64(*s["x"])[s["src"].long() // c["K"]]
        return torch.stack([s["dy"][a:b].double().t() @ x[a:b] for a, b in spans])
    g = torch.cat([s["dy"][a:b].double() @ s["w2"][e].double() for e, (a, b) in enumerate(spans)])
    h = _values64(*s["h"]).requires_grad_(True)
    gate, up = h[:, :c["H"]], h[:, c["H"]:]
    if c["limit"]:
        gate, up = gate.clamp(max=c["limit"]), up.clamp(-c["limit"], c["limit"])
    a = torch.nn.functional.silu(gate) * up
    (dh,) = torch.autograd.grad(a, h, g)
    return dh, a.detach()
