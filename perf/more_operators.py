"""Measured operators of serving the MoE path to a few tokens at a time: the whole
layer (router, experts, combine, shared expert) for at most 64 tokens, with bf16
or 4-bit expert weights; products of a few rows with 4-bit weights, dense or
grouped by expert; and the packing of weights to 4 bits and back.

A case is a dict of plain values; ``kind`` names the operator:

  layer      logits = bf16(x . w_router^T); scores by softmax or sigmoid, the top
             K of scores + bias; out = sum_k score * swiglu(x . w13[e]^T) . w2[e]^T
             (+ gate * the shared expert); ``bits`` of the expert weights: 16 or 4
  product    rows x times 4-bit weights, y = x . w^T; with ``E`` the rows lie in
             runs by expert
  store      bf16 weights packed to 4 bits and restored: what a packed weight is

4-bit weights are e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign) with one
power-of-two scale, a byte e + 127, for each 32 values along a row.  They are
laid out for 16-row tiles: codes [NB, C, 64, 16], exponents [NB, ceil(C / 4),
64, 4], NB = ceil(N / 16), C = ceil(K / 128).  Place l of a tile is row l % 16 and
columns 32 (l / 16) .. + 31 of 128; byte b holds columns 2 b (low half) and 2 b + 1.

``own`` chooses between the plain form (torch operations in 32 bits; the routing
in 64, where two candidates may lie close) and the framework's calls.
"""
from __future__ import annotations

import importlib
import math

import torch

own = False

_PKG = "torchtitan-ascend_amd"
_DEV = "cuda"
_BF16 = torch.bfloat16
_NORM_EPS = 1e-20
_GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _layer(T, E, K, D, H, bits, **o):
    return dict(dict(kind="layer", T=T, E=E, K=K, D=D, H=H, bits=bits, func="softmax", renorm=True, scale=1.0,
                     bias=False, before=False, limit=0.0, shared=0, gated=False), **o)


def _product(M, N, K, E=0, **o):
    return dict(dict(kind="product", M=M, N=N, K=K, E=E, skew=0.5, bias=False), **o)


def listed():
    cases = [
        # one sequence decoding through a layer of 128 small experts, eight per token
        ("layer_1_of_128", _layer(1, 128, 8, 2048, 768, 16)),
        # a decode batch of the same layer: most experts are hit, by two tokens each
        ("layer_32_of_128", _layer(32, 128, 8, 2048, 768, 16)),
        # five sequences through 16 large experts, one per token, and a shared one
        ("layer_5_of_16_shared", _layer(5, 16, 1, 5120, 8192, 16, func="sigmoid", renorm=False, shared=8192)),
        # a ragged batch of the debug model: the smallest weights, latency alone
        ("layer_61_of_8_debug", _layer(61, 8, 1, 256, 512, 16, func="sigmoid", renorm=False)),
        # one sequence decoding with 4-bit experts
        ("layer4_1_of_128", _layer(1, 128, 8, 2048, 768, 4)),
        # a full decode batch over a shard of 32 wide experts in 4 bits, with a gated shared expert
        ("layer4_64_of_32_shared", _layer(64, 32, 8, 7168, 2048, 4, func="sigmoid", scale=2.5, bias=True, shared=2048,
                                          gated=True)),
        # odd sizes: clamped activation, scores applied in front of the experts
        ("layer4_17_of_60_odd", _layer(17, 60, 4, 1440, 544, 4, before=True, limit=1.5, renorm=False)),
        # one token's down projection of a wide dense FFN
        ("product_1_5120x8192", _product(1, 5120, 8192)),
        # a short ragged batch through a projection whose sizes fill no tile
        ("product_13_1000x1440", _product(13, 1000, 1440, bias=True)),
        # a decode batch's rows in runs by expert, many experts without one
        ("product_96_128x1536x2048", _product(96, 1536, 2048, E=128)),
        # a small expert's weights of odd sizes
        ("store_1000x1440", dict(kind="store", E=1, N=1000, K=1440)),
        # a layer's whole w13, packed once when a model is loaded
        ("store_128x1536x2048", dict(kind="store", E=128, N=1536, K=2048)),
    ]
    return [dict(c, name=n) for n, c in cases]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    kind = rng.choice(["layer", "layer", "layer", "product", "product", "store"])
    if kind == "layer":
        E = rng.choice([4, 8, 16, 60, 64, 128])
        K = rng.randint(1, min(8, E))
        D, H = 32 * _log_int(rng, 4, 64), 32 * _log_int(rng, 4, 24)
        shared = rng.choice([0, 0, H, 32 * _log_int(rng, 4, 48)])
        return _layer(_log_int(rng, 1, 64), E, K, D, H, rng.choice([16, 4]), func=rng.choice(["softmax", "sigmoid"]),
                      renorm=rng.random() < 0.6, scale=rng.choice([1.0, 2.5]), bias=rng.random() < 0.4,
                      before=rng.random() < 0.3, limit=rng.choice([0.0, 0.0, 1.5]), shared=shared,
                      gated=shared > 0 and rng.random() < 0.5)
    if kind == "product":
        E = rng.choice([0, 0, 4, 32, 128])
        return _product(_log_int(rng, 1, 200), _log_int(rng, 64, 2048 if E else 8192), 32 * _log_int(rng, 2, 64), E=E,
                        skew=rng.choice([0.0, 0.5, 1.0]), bias=E == 0 and rng.random() < 0.5)
    return dict(kind="store", E=rng.choice([1, 3, 16]), N=_log_int(rng, 16, 4096), K=32 * _log_int(rng, 2, 128))


# ---------------------------------------------------------------------------
# 4-bit weights
# ---------------------------------------------------------------------------
def _pack_plain(w):
    """(codes, exponents) of weights [E, N, K] in the tiled layout: the smallest power of two 2^e with max|v| <= 6 * 2^e
    over each 32 values, codes nearest, ties to the even one."""
    E, N, K = w.shape
    nb, nc = (N + 15) // 16, (K + 127) // 128
    v = torch.nn.functional.pad(w.float(), (0, nc * 128 - K, 0, nb * 16 - N)).view(E, nb, 16, nc, 4, 32)
    v = v.permute(0, 1, 3, 4, 2, 5).reshape(E, nb, nc, 64, 32)  # a place's 32 columns together
    m, e = torch.frexp(v.abs().amax(4))  # absmax = m 2^e, 0.5 <= m < 1; 6 = 0.75 * 2^3
    e = (e - 3 + (m > 0.75).int()).clamp(-126, 125)
    e = torch.where(m == 0, torch.full_like(e, -126), e)
    a = torch.ldexp(v.abs(), -e.unsqueeze(4))
    # magnitudes up to 2 lie half a unit apart, up to 4 one, above that two
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    r = torch.round(a / step) * step
    code = torch.where(r < 2, r * 2, torch.where(r < 4, r + 2, r / 2 + 4)).to(torch.uint8).clamp(max=7)
    code = code + 8 * torch.signbit(v).to(torch.uint8)
    codes = code[..., 0::2] + 16 * code[..., 1::2]
    exps = torch.nn.functional.pad((e + 127).to(torch.uint8), (0, 0, 0, -nc % 4), value=127)
    return codes.contiguous(), exps.view(E, nb, (nc + 3) // 4, 4, 64).transpose(3, 4).contiguous()


def _unpack_plain(codes, exps, N, K):
    """fp32 values [E, N, K] of tiled 4-bit weights."""
    E, nb, nc = codes.shape[:3]
    grid = torch.tensor(_GRID, device=codes.device)
    grid = torch.cat([grid, -grid])
    half = torch.stack([codes & 15, codes >> 4], 5).view(E, nb, nc, 64, 32)
    e = exps.transpose(3, 4).reshape(E, nb, -1, 64)[:, :, :nc].int() - 127
    v = torch.ldexp(grid[half.int()], e.unsqueeze(4)).view(E, nb, nc, 4, 16, 32)
    return v.permute(0, 1, 4, 2, 3, 5).reshape(E, nb * 16, nc * 128)[:, :N, :K]


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _counts(case):
    """Rows per expert of a grouped product: a power law over experts in a fixed shuffled order."""
    E, M = case["E"], case["M"]
    w = [(i + 1) ** -case["skew"] for i in range(E)]
    c = [int(M * x / sum(w)) for x in w]
    for i in range(M - sum(c)):
        c[i % E] += 1
    order = torch.randperm(E, generator=torch.Generator().manual_seed(E)).tolist()
    return [c[i] for i in order]


def prepare(case, seed):
    gen = torch.Generator(device=_DEV)
    gen.manual_seed(seed)

    def normal(*shape, std=1.0, dtype=_BF16):
        return (torch.randn(*shape, generator=gen, device=_DEV) * std).to(dtype)

    def weights(E, N, K, bits):
        """bf16 [E, N, K], or the tiled pair of its 4-bit form."""
        if bits == 16:
            return torch.cat([normal(1, N, K, std=0.02) for _ in range(E)])
        parts = [_pack_plain(normal(1, N, K, std=0.02)) for _ in range(E)]
        return tuple(torch.cat([p[i] for p in parts]) for i in range(2))

    kind = case["kind"]
    s = dict(case=case)
    if kind == "layer":
        T, E, D, H, bits = (case[k] for k in ("T", "E", "D", "H", "bits"))
        s["x"] = normal(T, D)
        s["w_router"] = normal(E, D, std=0.02)
        s["bias"] = normal(E, std=0.05, dtype=torch.float32) if case["bias"] else None
        s["w13"] = weights(E, 2 * H, D, bits)
        s["w2"] = weights(E, D, H, bits)
        if case["shared"]:
            s["shared13"] = weights(1, 2 * case["shared"], D, bits)
            s["shared2"] = weights(1, D, case["shared"], bits)
            s["gate"] = normal(1, D, std=0.02) if case["gated"] else None
    elif kind == "product":
        s["x"] = normal(case["M"], case["K"])
        s["w"] = weights(max(case["E"], 1), case["N"], case["K"], 4)
        s["bias"] = normal(case["N"]) if case["bias"] else None
        s["offs"] = torch.tensor(_counts(case), device=_DEV).cumsum(0).int() if case["E"] else None
    else:
        s["w"] = normal(case["E"], case["N"], case["K"], std=0.02)
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    decode = importlib.import_module(_PKG + ".decode")
    c = s["case"]
    if c["kind"] == "store":
        return decode.unpack_e2m1(decode.pack_e2m1(s["w"]))
    if c["kind"] == "product":
        w = decode.PackedWeights(*s["w"], c["N"], c["K"])
        return decode.grouped_mm_e2m1(s["x"], w, s["offs"], bias=s["bias"])
    D, H, Hs = c["D"], c["H"], c["shared"]

    def weights(name, N, K):
        w = s.get(name)
        return decode.PackedWeights(*w, N, K) if isinstance(w, tuple) else w

    return decode.moe_decode(
        s["x"], s["w_router"], weights("w13", 2 * H, D), weights("w2", D, H), c["K"], c["func"], c["renorm"], c["scale"],
        s["bias"], _NORM_EPS, score_before_experts=c["before"], swiglu_limit=c["limit"] or None,
        shared_w13=weights("shared13", 2 * Hs, D), shared_w2=weights("shared2", D, Hs), shared_gate=s.get("gate"))


def _plain(s):
    return {"layer": _plain_layer, "product": _plain_product, "store": _plain_store}[s["case"]["kind"]](s)


def _wide(w, N, K):
    """fp32 [E, N, K] of bf16 weights or of a tiled 4-bit pair."""
    return _unpack_plain(*w, N, K) if isinstance(w, tuple) else w.float()


def _picked(w, at):
    return tuple(t[at] for t in w) if isinstance(w, tuple) else w[at]


def _route(s):
    """(scores fp32 [T, K], idx int64 [T, K]) in 64 bits from the bf16 logits."""
    c = s["case"]
    z = (s["x"].double() @ s["w_router"].double().t()).to(_BF16).double()
    if c["func"] == "softmax":
        ex = torch.exp(z - z.amax(1, keepdim=True))
        p = ex / ex.sum(1, keepdim=True)
    else:
        p = 1.0 / (1.0 + torch.exp(-z))
    v = p if s["bias"] is None else p + s["bias"].double()
    idx = torch.sort(v, dim=1, descending=True, stable=True).indices[:, :c["K"]].contiguous()
    w = p.gather(1, idx)
    if c["renorm"]:
        w = w / (w.sum(1, keepdim=True) + _NORM_EPS)
    return (w * c["scale"]).float(), idx


def _ffn(x, w13, w2, limit, score=None):
    """w2 . swiglu(w13 . x) with x [E, D, n], the products in 32 bits; score multiplies the first product."""
    h = torch.matmul(w13, x)
    if score is not None:
        h = h * score
    gate, up = h.chunk(2, 1)
    if limit:
        gate, up = gate.clamp(max=limit), up.clamp(-limit, limit)
    return torch.matmul(w2, gate / (1.0 + torch.exp(-gate)) * up)


def _plain_layer(s):
    c = s["case"]
    T, E, K, D, H, limit = (c[k] for k in ("T", "E", "K", "D", "H", "limit"))
    scores, idx = _route(s)
    x = s["x"].float()
    after = torch.ones_like(scores) if c["before"] else scores
    if T * K <= E:  # each choice takes its expert's weights
        at = idx.reshape(-1)
        first = scores.view(-1, 1, 1) if c["before"] else None
        y = _ffn(x.repeat_interleave(K, 0).unsqueeze(2), _wide(_picked(s["w13"], at), 2 * H, D),
                 _wide(_picked(s["w2"], at), D, H), limit, first).view(T, K, D)
    else:  # every token through every expert, then its choices
        w13, w2 = _wide(s["w13"], 2 * H, D), _wide(s["w2"], D, H)
        first = None
        if c["before"]:
            first = torch.zeros(E, T, device=x.device).scatter_(0, idx.t().contiguous(), scores.t().contiguous())
            first = first.unsqueeze(1)
        y = _ffn(x.t().contiguous().expand(E, D, T), w13, w2, limit, first)
        y = y[idx, :, torch.arange(T, device=x.device).unsqueeze(1)]
    out = (y * after.unsqueeze(2)).sum(1)
    if c["shared"]:
        Hs = c["shared"]
        sh = _ffn(x.t().contiguous().unsqueeze(0), _wide(s["shared13"], 2 * Hs, D), _wide(s["shared2"], D, Hs), limit)
        g = 1.0
        if s["gate"] is not None:
            z = (s["x"].double() @ s["gate"].double().t()).to(_BF16).float()
            g = 1.0 / (1.0 + torch.exp(-z))
        out = out + g * sh[0].t()
    return out.to(_BF16), scores, idx


def _plain_product(s):
    c = s["case"]
    w = _wide(s["w"], c["N"], c["K"])
    xt = s["x"].float().t().contiguous()
    if not c["E"]:
        y = torch.matmul(w[0], xt).t()
        return (y if s["bias"] is None else y + s["bias"].float()).to(_BF16)
    at = torch.arange(c["M"], device=xt.device)
    expert = torch.searchsorted(s["offs"].long(), at, right=True)
    return torch.matmul(w, xt.expand(c["E"], c["K"], c["M"]))[expert, :, at].to(_BF16)


def _plain_store(s):
    return _unpack_plain(*_pack_plain(s["w"]), s["case"]["N"], s["case"]["K"]).to(_BF16)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def _weight_bytes(N, K, bits):
    return 2 * N * K if bits == 16 else N * K / 2 + N * K / 32


def work(case):
    kind = case["kind"]
    if kind == "layer":
        T, E, K, D, H, Hs = (case[k] for k in ("T", "E", "K", "D", "H", "shared"))
        hit = E * (1.0 - (1.0 - K / E) ** T)  # experts that T tokens' choices reach on average
        b = 4 * T * D + 2 * E * D + 12 * T * K + 4 * E * case["bias"] + 2 * D * case["gated"]
        for n, h in ((hit, H), (1, Hs)):
            b += n * (_weight_bytes(2 * h, D, case["bits"]) + _weight_bytes(D, h, case["bits"]))
        return {"bytes": b, "flops": 2 * T * E * D + 6 * T * D * (K * H + Hs)}
    if kind == "product":
        M, N, K = case["M"], case["N"], case["K"]
        hit = sum(n > 0 for n in _counts(case)) if case["E"] else 1
        b = 2 * M * (N + K) + hit * _weight_bytes(N, K, 4) + 4 * case["E"] + 2 * N * case["bias"]
        return {"bytes": b, "flops": 2 * M * N * K}
    n = case["E"] * case["N"] * case["K"]
    return {"bytes": 4 * n, "flops": 0}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"layer": _exact_layer, "product": _exact_product, "store": _exact_store}[case["kind"]](s)


def _values64(w, e, N, K):
    """Expert e's weights in 64 bits: of a tiled pair, value (n, k) from its place in the tiles."""
    if not isinstance(w, tuple):
        return w[e].double()
    codes, exps = w[0][e], w[1][e]
    n, k = torch.arange(N, device=codes.device).unsqueeze(1), torch.arange(K, device=codes.device).unsqueeze(0)
    tile, chunk, place = n // 16, k // 128, n % 16 + 16 * (k % 128 // 32)
    code = (codes[tile, chunk, place, k % 32 // 2].int() >> (4 * (k % 2))) & 15
    mag, power = code & 7, (code & 7) >> 1
    # e2m1: exponents 1 to 3 hold 1.m, exponent 0 holds 0.m of the least
    val = torch.where(power > 0, (2 + mag % 2).double() * torch.exp2(power.double() - 2), 0.5 * mag.double())
    val = torch.where(code >= 8, -val, val)
    return val * torch.exp2(exps[tile, chunk // 4, place, chunk % 4].double() - 127)


def _exact_layer(s):
    c = s["case"]
    D, H = c["D"], c["H"]
    _, idx = _route(s)  # the selection; the values below are computed apart
    z = torch.nn.functional.linear(s["x"].double(), s["w_router"].double()).to(_BF16).double()
    p = torch.softmax(z, 1) if c["func"] == "softmax" else torch.sigmoid(z)
    scores = torch.gather(p, 1, idx)
    if c["renorm"]:
        scores = scores / scores.sum(1, keepdim=True)
    scores = scores * c["scale"]
    x = s["x"].double()
    out = torch.zeros(c["T"], D, dtype=torch.float64, device=x.device)

    def expert(rows, w13, w2, h, e):
        both = rows @ _values64(w13, e, 2 * h, D).t()
        gate, up = both[:, :h], both[:, h:]
        if c["limit"]:
            gate, up = gate.clamp(max=c["limit"]), up.clamp(-c["limit"], c["limit"])
        return (torch.nn.functional.silu(gate) * up) @ _values64(w2, e, D, h).t()

    for e in idx.unique().tolist():
        t, k = torch.nonzero(idx == e, as_tuple=True)
        score = scores[t, k].unsqueeze(1)
        if c["before"]:
            y = expert(x[t] * score, s["w13"], s["w2"], H, e)
        else:
            y = expert(x[t], s["w13"], s["w2"], H, e) * score
        out.index_add_(0, t, y)
    if c["shared"]:
        y = expert(x, s["shared13"], s["shared2"], c["shared"], 0)
        if s["gate"] is not None:
            y = y * torch.sigmoid((x @ s["gate"].double().t()).to(_BF16).double())
        out += y
    return out, scores, None


def _exact_product(s):
    c = s["case"]
    x = s["x"].double()
    if not c["E"]:
        y = x @ _values64(s["w"], 0, c["N"], c["K"]).t()
        return y if s["bias"] is None else y + s["bias"].double()
    ends = s["offs"].tolist()
    return torch.cat([x[a:b] @ _values64(s["w"], e, c["N"], c["K"]).t()
                      for e, (a, b) in enumerate(zip([0] + ends[:-1], ends))])


def _exact_store(s):
    """Each 32 values divided by the power of two found as a logarithm, and taken to the nearest of the 8 magnitudes by
    comparing with the midpoints between them; a midpoint goes to the code that is even."""
    w = s["w"]
    E, N, K = w.shape
    mid = [(a + b) / 2 for a, b in zip(_GRID, _GRID[1:])]
    out = []
    for e in range(E):
        v = w[e].double().view(N, K // 32, 32)
        most = v.abs().amax(2, keepdim=True)
        scale = torch.exp2(torch.ceil(torch.log2(most / 6.0)).clamp(-126, 125))
        a = v.abs() / scale
        r = torch.zeros_like(a)
        for i, m in enumerate(mid):
            above = a >= m if i % 2 else a > m  # code i + 1 is even for odd i
            r = torch.where(above, torch.full_like(r, _GRID[i + 1]), r)
        out.append((r * scale * torch.sign(v)).view(N, K))
    return torch.stack(out)
