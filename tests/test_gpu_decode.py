"""The MoE layer for a few tokens, products with 4-bit weights and their packing,
against the definitions in 64 bits.

Bounds are per element and derived.  A bf16 rounding moves a value by at most
2^-8 of it, a sum of n fp32 products by at most (n + 8) 2^-24 of the sum of
their sizes.  The activation is rounded once, so with dg and du the sums' errors
  |a - a'| <= (2^-8 + 2^-20) |a| + 1.1 |u| dg + |silu(g)| du + 1.1 dg du
(|silu'| < 1.1; 2^-20 for the fp32 sigmoid), and the output, with S = sum_k |s_k|
|w2| |a| and B the same sum over the bounds of a,
  |y - y'| <= 2^-8 |y| + (1 + 2^-8) (B + (H + K + 8) 2^-24 S).
Routing weights are fp32 roundings of 64-bit values: 2^-20 covers them and the
fp32 gate of the shared expert."""
from __future__ import annotations

import importlib

import numpy as np
import pytest
import torch

from gpu_util import DEV, announce

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


@pytest.fixture(scope="module")
def decode():
    return importlib.import_module("torchtitan-ascend_amd.decode")


def define_pack(w):
    """(values, exponent bytes [.., N, K / 32]) of weights by the definition."""
    w = np.asarray(w, np.float64)
    v = w.reshape(*w.shape[:-1], -1, 32)
    fin = np.isfinite(v)
    most = np.where(fin, np.abs(v), 0).max(-1, keepdims=True)
    with np.errstate(divide="ignore"):
        e = np.clip(np.ceil(np.log2(most / 6.0)), -126, 125)
    a = np.minimum(np.where(fin, np.abs(v), 0) / np.exp2(e), 6.0)
    step = np.where(a < 2, 0.5, np.where(a < 4, 1.0, 2.0))
    val = np.copysign(np.round(a / step) * step * np.exp2(e), v)
    bad = ~fin.all(-1, keepdims=True)
    return (np.where(bad, np.nan, val).reshape(w.shape),
            np.where(bad, 255, e + 127)[..., 0].astype(np.int64))


def from_tiles(p):
    """(values, exponent bytes) of packed weights, place by place."""
    codes, exps = p.codes.cpu().numpy(), p.exponents.cpu().numpy()
    n, k = np.arange(p.rows)[:, None], np.arange(p.cols)[None, :]
    place = n % 16 + 16 * (k % 128 // 32)
    byte = codes[:, n // 16, k // 128, place, k % 32 // 2].astype(np.int64)
    code = byte >> (4 * (k % 2)) & 15
    e = exps[:, n // 16, k // 512, place, k // 128 % 4].astype(np.int64)
    v = GRID[code & 7] * np.exp2(e.astype(np.float64) - 127)
    return np.where(e == 255, np.nan, np.where(code > 7, -v, v)), e[:, :, ::32]


def weights(rng, *shape, scale=0.05):
    return torch.from_numpy(rng.standard_normal(shape) * scale).to(BF16).to(DEV)


# ---------------------------------------------------------------------------
# 4-bit weights
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("E,N,K", [(1, 1, 32), (1, 16, 128), (3, 17, 160), (2, 100, 544), (1, 1000, 1440),
                                   (5, 48, 2048), (1, 33, 96), (2, 15, 1056)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_pack_and_restore(decode, E, N, K, dtype):
    rng = np.random.default_rng(E + N + K)
    w = rng.standard_normal((E, N, K)) * np.exp2(rng.integers(-20, 20, (E, N, 1)) + rng.standard_normal((1, 1, K)))
    w = torch.from_numpy(w).to(dtype).to(DEV)
    announce(f"pack_e2m1 E={E} N={N} K={K} {dtype}")
    p = decode.pack_e2m1(w)
    y = decode.unpack_e2m1(p)
    torch.cuda.synchronize()
    val, e = define_pack(w.double().cpu().numpy())
    got, ge = from_tiles(p)
    np.testing.assert_array_equal(ge, e)
    np.testing.assert_array_equal(got, val)
    np.testing.assert_array_equal(y.double().cpu().numpy(), val)
    # restored weights pack to themselves
    assert torch.equal(decode.unpack_e2m1(decode.pack_e2m1(y)), y)


def test_pack_special_values(decode):
    """Ends of the range, exponent borders, ties, zeros of both signs, subnormal
    groups, NaN and infinities."""
    x = np.zeros((12, 64))
    x[1, :] = -0.0
    x[2, :4] = [3.3895e38, -3.3895e38, 1.0, 2.0 ** 125]
    x[3, :3] = [6.0, 6.03125, 1.0]
    x[3, 32:35] = [6.03125, 3.0, 0.1]
    x[4, :8] = [6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    x[5, :8] = [-6.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0]
    x[6, :3] = [2.0 ** -126, 2.0 ** -127, -2.0 ** -130]
    x[7, :2] = [np.nan, 1.0]
    x[8, 40] = np.inf
    x[9, :] = -np.inf
    x[10, 63] = -2.0 ** 100
    x[11, :4] = [4.0, 0.125, 0.3125, 0.3]
    t = torch.from_numpy(x).to(BF16).to(DEV)
    p = decode.pack_e2m1(t)
    y = decode.unpack_e2m1(p)
    val, e = define_pack(t.double().cpu().numpy()[None])
    got, ge = from_tiles(p)
    np.testing.assert_array_equal(ge, e)
    np.testing.assert_array_equal(got, val)
    np.testing.assert_array_equal(y.double().cpu().numpy(), val)


def test_every_code_at_every_exponent(decode):
    """Row-major codes of all 16 values at all 256 exponent bytes, tiled and restored:
    code * 2^(byte - 127) rounded to bf16 (past its range an infinity), byte 255 NaN."""
    pair = torch.arange(16, dtype=torch.uint8)
    codes = (pair + 16 * pair.flip(0)).repeat(256, 1).contiguous()  # [256, 16]: K = 32
    exps = torch.arange(256, dtype=torch.uint8).view(256, 1)
    p = decode.tile_e2m1(codes.to(DEV), exps.to(DEV))
    y = decode.unpack_e2m1(p)[0].double().cpu()
    low, high = codes.long() & 15, codes.long() >> 4
    c = torch.stack([low, high], 2).view(256, 32)
    v = torch.from_numpy(GRID)[c & 7] * torch.exp2(exps.double() - 127)
    v = torch.where(c > 7, -v, v).float().to(BF16).double()
    v[255] = float("nan")
    np.testing.assert_array_equal(y.numpy(), v.numpy())


@pytest.mark.parametrize("E,N,K", [(1, 5, 32), (2, 40, 672), (1, 16, 512)])
def test_tile_of_row_major_codes(decode, E, N, K):
    rng = np.random.default_rng(K)
    codes = torch.from_numpy(rng.integers(0, 256, (E, N, K // 2), dtype=np.uint8)).to(DEV)
    exps = torch.from_numpy(rng.integers(110, 140, (E, N, K // 32), dtype=np.uint8)).to(DEV)
    got, e = from_tiles(decode.tile_e2m1(codes, exps))
    np.testing.assert_array_equal(e, exps.cpu().numpy())
    c = codes.cpu().numpy().astype(np.int64)
    c = np.stack([c & 15, c >> 4], -1).reshape(E, N, K)
    v = GRID[c & 7] * np.exp2(exps.cpu().numpy().astype(np.float64) - 127).repeat(32, -1)
    np.testing.assert_array_equal(got, np.where(c > 7, -v, v))


# ---------------------------------------------------------------------------
# Products with 4-bit weights
# ---------------------------------------------------------------------------
def check_product(x, w, y, bias=None):
    x, w, y = x.double(), w.double(), y.double()
    ref, size = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        ref, size = ref + bias.double(), size + bias.double().abs()
    bound = 2.0 ** -8 * ref.abs() + (1 + 2.0 ** -8) * (x.shape[1] + 9) * 2.0 ** -24 * size
    off = (y - ref).abs() - bound
    assert off.max() <= 0, f"{off.max().item():.3e} past the bound"


@pytest.mark.parametrize("M,N,K", [(1, 1, 32), (1, 16, 32), (1, 5120, 8192), (2, 31, 96), (7, 33, 288), (13, 1000, 1440),
                                   (16, 2048, 2048), (17, 130, 544), (40, 64, 2080), (64, 96, 4096), (65, 257, 160),
                                   (200, 1003, 1024), (1000, 40, 256)])
@pytest.mark.parametrize("bias", [None, torch.bfloat16, torch.float32])
def test_dense_product(decode, M, N, K, bias):
    rng = np.random.default_rng(M + N + K)
    x, p = weights(rng, M, K, scale=1.0), decode.pack_e2m1(weights(rng, N, K))
    b = None if bias is None else torch.randn(N, device=DEV).to(bias)
    announce(f"grouped_mm_e2m1 dense M={M} N={N} K={K} bias={bias}")
    y = decode.grouped_mm_e2m1(x, p, bias=b)
    check_product(x, decode.unpack_e2m1(p)[0], y, b)
    assert torch.equal(y, decode.grouped_mm_e2m1(x, p, bias=b))


@pytest.mark.parametrize("counts,N,K", [([1], 40, 64), ([0, 3, 0, 1], 96, 1056), ([5, 0, 17, 64, 65, 2], 130, 512),
                                        ([0, 0, 0], 32, 32), ([1] * 60, 1536, 2048), ([200, 1, 300], 31, 160)])
@pytest.mark.parametrize("past", [0, 5])
def test_grouped_product(decode, counts, N, K, past):
    """Rows in runs by expert, with `past` rows behind the last run: left as they were."""
    rng = np.random.default_rng(sum(counts) + N)
    M, E = sum(counts) + past, len(counts)
    x, p = weights(rng, M, K, scale=1.0), decode.pack_e2m1(weights(rng, E, N, K))
    offs = torch.tensor(counts, device=DEV).cumsum(0).int()
    announce(f"grouped_mm_e2m1 counts={counts[:8]} N={N} K={K} past={past}")
    y = decode.grouped_mm_e2m1(x, p, offs)
    w, r = decode.unpack_e2m1(p), 0
    for e, c in enumerate(counts):
        if c:
            check_product(x[r:r + c], w[e], y[r:r + c])
        r += c
    if M == 0:
        assert y.shape == (0, N)


# ---------------------------------------------------------------------------
# The layer
# ---------------------------------------------------------------------------
def layer_ref(x, scores, idx, w13, w2, before, limit, shared=None, gate=None):
    """(output, bound) in 64 bits; weights as bf16 tensors."""
    T, D = x.shape
    E, H = w13.shape[0], w13.shape[1] // 2
    K = idx.shape[1]
    x = x.double()
    out = torch.zeros(T, D, dtype=torch.float64, device=x.device)
    bound, size = torch.zeros_like(out), torch.zeros_like(out)

    def ffn(rows, a13, a2, h, factor):
        a13, a2 = a13.double(), a2.double()
        z = rows @ a13.t() * factor
        dz = (D + 9) * 2.0 ** -24 * (rows.abs() @ a13.abs().t()) * factor.abs()
        g, u, dg, du = z[:, :h], z[:, h:], dz[:, :h], dz[:, h:]
        if limit is not None:
            g, u = g.clamp(max=limit), u.clamp(-limit, limit)
        s = g * torch.sigmoid(g)
        a = s * u
        da = (2.0 ** -8 + 2.0 ** -20) * a.abs() + 1.1 * u.abs() * dg + s.abs() * du + 1.1 * dg * du
        return a @ a2.t(), da @ a2.abs().t(), a.abs() @ a2.abs().t()

    one = torch.ones(1, 1, dtype=torch.float64, device=x.device)
    for e in range(E):
        t, k = torch.nonzero(idx == e, as_tuple=True)
        if not len(t):
            continue
        sc = scores[t, k].double().unsqueeze(1)
        y, dy, sy = ffn(x[t], w13[e], w2[e], H, sc if before else one)
        m = one if before else sc
        out.index_add_(0, t, y * m)
        bound.index_add_(0, t, dy * m.abs())
        size.index_add_(0, t, sy * m.abs())
    if shared is not None:
        y, dy, sy = ffn(x, shared[0], shared[1], shared[0].shape[0] // 2, one)
        m = one if gate is None else gate.double().view(T, 1)
        out, bound, size = out + y * m, bound + dy * m, size + sy * m
    n = max(H, 0 if shared is None else shared[1].shape[1]) + K + 9
    return out, 2.0 ** -8 * out.abs() + (1 + 2.0 ** -8) * (bound + (n * 2.0 ** -24 + 2.0 ** -20) * size)


def build(decode, rng, E, D, H, bits, shared=0):
    """(weights to pass, the bf16 weights they stand for)."""
    pairs = [weights(rng, E, 2 * H, D), weights(rng, E, D, H)]
    if shared:
        pairs += [weights(rng, 2 * shared, D), weights(rng, D, shared)]
    if bits == 16:
        return pairs, pairs
    packed = [decode.pack_e2m1(w) for w in pairs]
    return packed, [decode.unpack_e2m1(p).view(w.shape) for p, w in zip(packed, pairs)]


LAYERS = [
    # T, E, K, D, H
    (1, 128, 8, 2048, 768),
    (1, 1, 1, 32, 32),
    (2, 4, 2, 160, 96),
    (5, 16, 1, 256, 512),
    (16, 8, 2, 1440, 544),
    (17, 60, 4, 96, 1056),
    (33, 3, 3, 512, 64),
    (61, 8, 1, 256, 512),
    (64, 2, 1, 2080, 288),
    (64, 128, 16, 128, 32),
]


@pytest.mark.parametrize("T,E,K,D,H", LAYERS)
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("form", ["plain", "before", "shared"])
def test_experts_stage(decode, T, E, K, D, H, bits, form):
    rng = np.random.default_rng(T * 7 + E + D + bits)
    Hs = 0 if form != "shared" else (H if D % 64 else 96)
    w, wb = build(decode, rng, E, D, H, bits, Hs)
    x = weights(rng, T, D, scale=1.0)
    idx = torch.from_numpy(np.argsort(rng.random((T, E)), axis=1)[:, :K].copy()).to(DEV)
    scores = torch.rand(T, K, device=DEV)
    scale = torch.rand(T, device=DEV) if Hs and T % 2 else None
    limit = 0.7 if form == "before" else None
    announce(f"experts_decode T={T} E={E} K={K} D={D} H={H} bits={bits} {form}")
    y = decode.experts_decode(x, scores, idx, *w[:2], form == "before", limit, *(w[2:] or (None, None)), scale)
    ref, bound = layer_ref(x, scores, idx, *wb[:2], form == "before", limit, wb[2:] or None, scale)
    off = ((y.double() - ref).abs() - bound).max().item()
    assert off <= 0, f"{off:.3e} past the bound"
    again = decode.experts_decode(x, scores, idx.int(), *w[:2], form == "before", limit, *(w[2:] or (None, None)), scale)
    assert torch.equal(y, again)


@pytest.mark.parametrize("bits", [16, 4])
def test_labels_that_repeat_or_name_no_expert(decode, bits):
    """The same expert twice for a token (all of a batch on one expert, more rows than a
    pass holds), labels outside [0, E), tokens and batches without any."""
    rng = np.random.default_rng(5)
    T, E, K, D, H = 64, 6, 8, 128, 64
    w, wb = build(decode, rng, E, D, H, bits)
    x, scores = weights(rng, T, D, scale=1.0), torch.rand(T, K, device=DEV)
    mixed = torch.from_numpy(rng.integers(-2, E + 2, (T, K))).to(DEV)
    mixed[3] = -1
    mixed[4] = E
    mixed[5] = 2 ** 40
    for name, idx in (("one expert", torch.full((T, K), 4, device=DEV)), ("mixed", mixed),
                      ("none", torch.full((T, K), -1, device=DEV))):
        announce(f"experts_decode labels {name} bits={bits}")
        y = decode.experts_decode(x, scores, idx, *w)
        ref, bound = layer_ref(x, scores, idx, *wb, False, None)
        assert ((y.double() - ref).abs() - bound).max() <= 0, name
        if name == "mixed":
            assert not y[3:6].any()
        if name == "none":
            assert not y.any()


@pytest.mark.parametrize("T,E,K,D", [(1, 128, 8, 2048), (1, 4, 1, 32), (3, 60, 4, 1440), (8, 16, 1, 5120), (9, 256, 8, 7168),
                                     (64, 160, 6, 128), (33, 1024, 16, 64)])
@pytest.mark.parametrize("func", ["softmax", "sigmoid"])
def test_router(decode, ops, T, E, K, D, func):
    """Logits from 64-bit sums, then the same picks and weights as the selection from
    given logits; the gate is the sigmoid of its bf16 product."""
    rng = np.random.default_rng(T + E)
    x, wr, wg = weights(rng, T, D, scale=1.0), weights(rng, E, D, scale=0.02), weights(rng, 1, D, scale=0.02)
    bias = torch.randn(E, device=DEV) * 0.05 if T % 2 else None
    announce(f"router_decode T={T} E={E} K={K} D={D} {func}")
    scores, idx, gate = decode.router_decode(x, wr, K, func, True, 2.5, bias, shared_gate=wg)
    z = (x.double() @ wr.double().t()).to(BF16)
    s2, i2 = ops.router_topk(z, K, func, True, 2.5, bias, num_groups=1, topk_groups=1)
    assert torch.equal(idx, i2) and torch.equal(scores, s2)
    g = torch.sigmoid((x.double() @ wg.double().t()).to(BF16).double())[:, 0]
    assert ((gate.double() - g).abs() <= 2.0 ** -20 * g).all()
    if E % 4 == 0 and K <= E // 2:
        s1, i1, none = decode.router_decode(x, wr, K, func, num_groups=4, topk_groups=2)
        s2, i2 = ops.router_topk(z, K, func, num_groups=4, topk_groups=2)
        assert none is None and torch.equal(i1, i2) and torch.equal(s1, s2)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("T,E,K,D,H", [(1, 128, 8, 2048, 768), (17, 60, 4, 1440, 544), (64, 8, 2, 256, 512),
                                       (3, 16, 2, 128, 96), (20, 160, 6, 64, 32), (64, 256, 8, 64, 32),
                                       (33, 1024, 16, 64, 32), (5, 300, 9, 32, 64), (40, 64, 12, 96, 32)])
def test_whole_layer(decode, T, E, K, D, H, bits):
    rng = np.random.default_rng(T)
    w, wb = build(decode, rng, E, D, H, bits, 96)
    x, wr, wg = weights(rng, T, D, scale=1.0), weights(rng, E, D, scale=0.02), weights(rng, 1, D, scale=0.02)
    announce(f"moe_decode T={T} E={E} K={K} D={D} H={H} bits={bits}")
    out, scores, idx = decode.moe_decode(x, wr, *w[:2], K, "softmax", True, shared_w13=w[2], shared_w2=w[3],
                                         shared_gate=wg)
    s, i, gate = decode.router_decode(x, wr, K, "softmax", True, shared_gate=wg)
    assert torch.equal(scores, s) and torch.equal(idx, i)
    assert torch.equal(out, decode.experts_decode(x, s, i, *w[:2], False, None, w[2], w[3], gate))
    ref, bound = layer_ref(x, s, i, *wb[:2], False, None, wb[2:], gate)
    assert ((out.double() - ref).abs() - bound).max() <= 0
    if E % 4 == 0 and K <= E // 2:
        groups = dict(num_groups=4, topk_groups=2, group_score="max")
        out, scores, idx = decode.moe_decode(x, wr, *w[:2], K, "sigmoid", **groups)
        s, i, _ = decode.router_decode(x, wr, K, "sigmoid", **groups)
        assert torch.equal(scores, s) and torch.equal(idx, i)
        assert torch.equal(out, decode.experts_decode(x, s, i, *w[:2]))


def test_without_tokens(decode):
    rng = np.random.default_rng(0)
    w, _ = build(decode, rng, 4, 64, 32, 16)
    x, wr = torch.empty(0, 64, dtype=BF16, device=DEV), weights(rng, 4, 64)
    out, scores, idx = decode.moe_decode(x, wr, *w, 2)
    assert out.shape == (0, 64) and scores.shape == idx.shape == (0, 2)
    assert decode.grouped_mm_e2m1(x, decode.pack_e2m1(weights(rng, 8, 64))).shape == (0, 8)
    assert decode.unpack_e2m1(decode.pack_e2m1(torch.empty(0, 8, 64, dtype=BF16, device=DEV))).shape == (0, 8, 64)
