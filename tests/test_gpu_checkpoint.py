"""8-bit activation checkpoints: packing and restoring against the definition in
64 bits (exactly), and the backward products that read packed rows against
the bf16 products on the restored rows (bit for bit: restored values are exact
in bf16, and the kernels then do the same arithmetic) and against 64 bits."""
from __future__ import annotations

import importlib

import numpy as np
import pytest
import torch

from gpu_util import DEV, announce, rel_err_rows, to_np, zipf_counts

BF16 = torch.bfloat16


def define(x):
    """(exponent bytes, values) of rows x (float64) by the definition: the block's power of two from a logarithm,
    values on the grid of 3 places below their own power of two, at least 2^-6."""
    x = np.asarray(x, np.float64)
    R, C = x.shape
    nb = (C + 127) // 128
    pad = np.zeros((R, nb * 128))
    pad[:, :C] = np.where(np.isfinite(x), np.abs(x), 0.0)
    most = pad.reshape(R, nb, 128).max(2)
    with np.errstate(divide="ignore"):
        e = np.clip(np.ceil(np.log2(most / 448.0)), -118, 120)
    s = np.exp2(e)[:, np.arange(C) // 128]
    with np.errstate(invalid="ignore"):
        v = x / s
        step = np.exp2(np.floor(np.log2(np.maximum(np.abs(v), 2.0 ** -6))) - 3)
        # at e = 120 codes end at 240: 256 * 2^120 = 2^128 is no bf16 number
        r = np.round(v / step) * step
        val = np.where(e[:, np.arange(C) // 128] == 120, np.clip(r, -240, 240), r) * s
    return (e + 127).astype(np.int64), np.where(np.isfinite(x), val, np.nan)


def rows(rng, R, C):
    """bf16 rows whose columns span many binades."""
    x = rng.standard_normal((R, C)) * np.exp2(rng.standard_normal((1, C)) * 4)
    return torch.from_numpy(x).to(BF16).to(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("R,C", [(1, 8), (3, 128), (1003, 1544), (5, 136), (4096, 1536), (2, 8192), (257, 120),
                                 (9000, 640), (1, 16384)])
def test_pack_and_restore(ops, R, C):
    rng = np.random.default_rng(R + C)
    x = rows(rng, R, C)
    announce(f"pack R={R} C={C}")
    p = ops.pack_e4m3(x)
    y = ops.unpack_e4m3(p)
    torch.cuda.synchronize()
    e, val = define(x.double().cpu().numpy())
    np.testing.assert_array_equal(p.exponents.cpu().numpy(), e)
    np.testing.assert_array_equal(y.double().cpu().numpy(), val)
    assert p.codes.shape == (R, C) and p.exponents.shape == (R, (C + 127) // 128)
    # packing restored rows gives the same values: the grid holds them
    again = ops.unpack_e4m3(ops.pack_e4m3(y))
    assert torch.equal(again, y)


@pytest.mark.gpu
def test_special_values(ops):
    """Zeros of both signs, the ends of bf16's range, borders of the exponent
    (448 * 2^e and the next bf16 value), ties, NaN and infinities beside
    finite values, blocks of nothing else."""
    x = np.zeros((12, 264), np.float64)
    x[1, :] = -0.0
    x[2, :3] = [3.3895e38, -3.3895e38, 1.0]
    x[3, :3] = [9.2e-41, -1.2e-38, 2.0 ** -120]
    x[4, :4] = [448.0, 450.0, 1.0, -0.3]
    x[5, 0], x[5, 128], x[5, 256] = 448.0, 450.0, 1.75
    x[6, :6] = [256.0, 17.0, 19.0, 0.0146484375, 0.0009765625, 0.00048828125]  # ties at 3 places, at 2^-9 and below
    x[7, :4] = [np.nan, 1.0, np.inf, -np.inf]
    x[7, 130] = 5.0
    x[8, :128] = np.nan
    x[9, :] = np.inf
    x[10, 263] = -2.0 ** 100
    x[11, 0] = 2.0 ** -112 * 1.875
    t = torch.from_numpy(x).to(BF16).to(DEV)
    p = ops.pack_e4m3(t)
    y = ops.unpack_e4m3(p)
    e, val = define(t.double().cpu().numpy())
    np.testing.assert_array_equal(p.exponents.cpu().numpy(), e)
    np.testing.assert_array_equal(y.double().cpu().numpy(), val)
    assert not ops.unpack_e4m3(ops.pack_e4m3(t[:2])).any()


@pytest.mark.gpu
@pytest.mark.parametrize("T,C,K", [(1, 256, 8), (300, 136, 8), (1000, 2048, 1)])
def test_unpack_gathered_and_scaled(ops, T, C, K):
    rng = np.random.default_rng(T + C)
    x = rows(rng, T, C)
    p = ops.pack_e4m3(x)
    y = ops.unpack_e4m3(p)
    src = torch.from_numpy(rng.permutation(T * K).astype(np.int32)).to(DEV)
    scale = torch.from_numpy(rng.random(T * K).astype(np.float32)).to(DEV)
    announce(f"unpack gathered T={T} C={C} K={K}")
    got = ops.unpack_e4m3(p, src, K)
    assert torch.equal(got, y[src.long() // K])
    got = ops.unpack_e4m3(p, src, K, scale)
    assert torch.equal(got, (y.float()[src.long() // K] * scale[:, None]).to(BF16))
    assert torch.equal(ops.unpack_e4m3(p, row_scale=scale[:T]), (y.float() * scale[:T, None]).to(BF16))
    # an index past the rows is clamped to them
    far = torch.tensor([0, T * K + 10 ** 6, -5], dtype=torch.int32, device=DEV)
    assert torch.equal(ops.unpack_e4m3(p, far, K), y[[0, T - 1, 0]])


@pytest.mark.gpu
def test_empty_strided_and_captured(ops):
    assert ops.unpack_e4m3(ops.pack_e4m3(torch.empty(0, 64, dtype=BF16, device=DEV))).shape == (0, 64)
    wide = torch.randn(50, 400, device=DEV).to(BF16)
    assert torch.equal(ops.unpack_e4m3(ops.pack_e4m3(wide[:, 5:141])),
                       ops.unpack_e4m3(ops.pack_e4m3(wide[:, 5:141].contiguous())))
    x = torch.randn(500, 264, device=DEV).to(BF16)
    ops.unpack_e4m3(ops.pack_e4m3(x))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ops.unpack_e4m3(ops.pack_e4m3(x))
    for _ in range(3):
        x.normal_()
        g.replay()
        want = ops.unpack_e4m3(ops.pack_e4m3(x))
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def offsets(counts):
    return torch.from_numpy(np.cumsum(counts).astype(np.int32)).to(DEV)


GEMMS = [
    # counts, D, H
    ([5], 128, 128),
    ([0, 1, 0, 63, 64, 65, 0], 192, 128),
    ([321, 0, 640, 31], 256, 384),
    ([0, 0, 0], 128, 128),
    ([700, 900], 512, 256),
    ([1] * 40, 256, 128),
]


@pytest.mark.gpu
@pytest.mark.parametrize("counts,D,H", GEMMS)
@pytest.mark.parametrize("limit", [None, 0.5])
def test_dgrad_swiglu_packed(ops, counts, D, H, limit):
    """Against the bf16 form on the restored h, bit for bit, and against 64
    bits: one rounding to bf16 (2^-8 of the value) and fp32 sums of D products
    (D 2^-24 of their sizes, far below) relative to the row's largest value,
    for which 2^-7 leaves a factor of two."""
    rng = np.random.default_rng(sum(counts) + D + H)
    M, E = sum(counts) + 7, len(counts)  # seven rows behind the last expert
    dy = torch.from_numpy(rng.standard_normal((M, D))).to(BF16).to(DEV)
    w2 = torch.from_numpy(rng.standard_normal((E, D, H)) * 0.05).to(BF16).to(DEV)
    h = ops.pack_e4m3(torch.from_numpy(rng.standard_normal((M, 2 * H))).to(BF16).to(DEV))
    offs = offsets(counts)
    announce(f"dgrad packed counts={counts} D={D} H={H} limit={limit}")
    dh, a = ops.grouped_mm_dgrad_swiglu_packed(dy, w2, h, offs, limit, want_a=True)
    hb = ops.unpack_e4m3(h)
    dh0, a0 = ops.grouped_mm_dgrad_swiglu(dy, w2, hb, offs, limit, want_a=True)
    torch.cuda.synchronize()
    n = sum(counts)
    assert torch.equal(dh[:n], dh0[:n]) and torch.equal(a[:n], a0[:n])
    if n == 0:
        return
    hd = hb[:n].double().requires_grad_(True)
    gate, up = hd[:, :H], hd[:, H:]
    if limit is not None:
        gate, up = gate.clamp(max=limit), up.clamp(-limit, limit)
    act = torch.nn.functional.silu(gate) * up
    e = np.repeat(np.arange(E), counts)
    g = torch.cat([dy[i:i + 1].double() @ w2[e[i]].double() for i in range(n)])
    (rdh,) = torch.autograd.grad(act, hd, g)
    assert rel_err_rows(to_np(dh[:n]), rdh.cpu().numpy()) < 2.0 ** -7
    assert rel_err_rows(to_np(a[:n]), act.detach().cpu().numpy()) < 2.0 ** -7
    # without a
    dh1, none = ops.grouped_mm_dgrad_swiglu_packed(dy, w2, h, offs, limit)
    assert none is None and torch.equal(dh1[:n], dh[:n])


@pytest.mark.gpu
def test_dgrad_rows_behind_the_last_expert_stay(ops):
    """Through the C ABI into given buffers: rows at and past offs[E - 1] are not written."""
    import ctypes

    L = importlib.import_module("torchtitan-ascend_amd._lib")
    rng = np.random.default_rng(3)
    M, D, H, n = 90, 128, 128, 70
    dy = torch.from_numpy(rng.standard_normal((M, D))).to(BF16).to(DEV)
    w2 = torch.from_numpy(rng.standard_normal((2, D, H)) * 0.05).to(BF16).to(DEV)
    h = ops.pack_e4m3(torch.from_numpy(rng.standard_normal((M, 2 * H))).to(BF16).to(DEV))
    offs = offsets([30, 40])
    dh = torch.full((M, 2 * H), 7.0, dtype=BF16, device=DEV)
    a = torch.full((M, H), 7.0, dtype=BF16, device=DEV)
    ws = torch.empty(L.load().ttamd_gemm_workspace_bytes(M, 2), dtype=torch.uint8, device=DEV)
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    L.call("ttamd_grouped_mm_dgrad_swiglu_packed", p(dy), p(w2), p(h.codes), p(h.exponents), p(offs), M, 2, D, H,
           float("nan"), p(dh), p(a), p(ws), ws.numel(), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert bool((dh[n:] == 7).all()) and bool((a[n:] == 7).all()) and not bool((dh[:n] == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("T,K,E,N,D,skew", [
    (1, 1, 1, 128, 128, 0.0), (37, 8, 16, 256, 128, 1.0), (500, 2, 3, 384, 640, 0.5), (640, 8, 20, 256, 512, 1.2),
    (3000, 1, 4, 128, 256, 0.0), (50, 4, 64, 128, 384, 0.0),
])
@pytest.mark.parametrize("dtype", [torch.float32, BF16])
def test_wgrad_packed(ops, T, K, E, N, D, skew, dtype):
    """Against the bf16 form on the restored, gathered rows: bit for bit, with
    and without a row scale; and the fp32 gradient against 64 bits: fp32 sums
    of the expert's rows, each term's rounding 2^-24 of its size and at most
    rows + 16 of them."""
    rng = np.random.default_rng(T + K + E)
    M = T * K
    counts = zipf_counts(M, E, skew, max(1, E - E // 4), rng)
    x = ops.pack_e4m3(torch.from_numpy(rng.standard_normal((T, D))).to(BF16).to(DEV))
    dy = torch.from_numpy(rng.standard_normal((M, N))).to(BF16).to(DEV)
    src = torch.from_numpy(rng.permutation(M).astype(np.int32)).to(DEV)
    scale = torch.from_numpy(rng.random(M).astype(np.float32)).to(DEV)
    offs = offsets(counts)
    announce(f"wgrad packed T={T} K={K} E={E} N={N} D={D} {dtype}")
    routed = ops.unpack_e4m3(x, src, K)
    got = ops.grouped_mm_wgrad_packed(dy, x, offs, E, dtype, src, K)
    want = ops.grouped_mm_wgrad(dy, routed, offs, E, dtype)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    got = ops.grouped_mm_wgrad_packed(dy, x, offs, E, dtype, src, K, scale)
    assert torch.equal(got, ops.grouped_mm_wgrad(dy, ops.unpack_e4m3(x, src, K, scale), offs, E, dtype))
    if K == 1:
        got = ops.grouped_mm_wgrad_packed(dy, x, offs, E, dtype)
        assert torch.equal(got, ops.grouped_mm_wgrad(dy, ops.unpack_e4m3(x), offs, E, dtype))
    if dtype == torch.float32:
        ends = np.cumsum(counts)
        for e in range(E):
            a, b = int(ends[e] - counts[e]), int(ends[e])
            ref = dy[a:b].double().t() @ routed[a:b].double()
            size = dy[a:b].double().abs().t() @ routed[a:b].double().abs()
            assert bool(((want[e].double() - ref).abs() <= size * (b - a + 16) * 2.0 ** -24).all())


@pytest.mark.gpu
def test_wgrad_packed_without_rows(ops):
    """No rows at all, and no rows of any expert: exact zeros."""
    x = ops.pack_e4m3(torch.randn(16, 128, device=DEV).to(BF16))
    none = torch.zeros(3, dtype=torch.int32, device=DEV)
    src = torch.zeros(0, dtype=torch.int32, device=DEV)
    announce("wgrad packed without rows")
    for dtype in (torch.float32, BF16):
        dw = ops.grouped_mm_wgrad_packed(torch.empty(0, 128, dtype=BF16, device=DEV), x, none, 3, dtype, src, 8)
        assert dw.shape == (3, 128, 128) and not dw.any()
        dy = torch.randn(16, 128, device=DEV).to(BF16)
        src16 = torch.arange(16, dtype=torch.int32, device=DEV)
        dw = ops.grouped_mm_wgrad_packed(dy, x, none, 3, dtype, src16, 1)
        assert not dw.any()


@pytest.mark.gpu
def test_wgrad_packed_same_token_everywhere(ops):
    """Every routed row the same token, and indices out of range (clamped)."""
    rng = np.random.default_rng(12)
    x = ops.pack_e4m3(torch.from_numpy(rng.standard_normal((5, 256))).to(BF16).to(DEV))
    dy = torch.from_numpy(rng.standard_normal((200, 128))).to(BF16).to(DEV)
    offs = offsets([90, 0, 110])
    for v, row in ((3, 3), (10 ** 6, 4), (-9, 0)):
        src = torch.full((200,), v, dtype=torch.int32, device=DEV)
        got = ops.grouped_mm_wgrad_packed(dy, x, offs, 3, torch.float32, src, 1)
        want = ops.grouped_mm_wgrad(dy, ops.unpack_e4m3(x)[row].expand(200, 256).contiguous(), offs, 3, torch.float32)
        assert torch.equal(got, want)


@pytest.mark.gpu
def test_wgrad_packed_large_gathered(ops):
    """Full rounds, a split tail and experts that end inside a stage."""
    rng = np.random.default_rng(9)
    T, K, E, N, D = 1024, 8, 24, 768, 1024
    M = T * K
    counts = zipf_counts(M, E, 0.8, 20, rng)
    x = ops.pack_e4m3(torch.from_numpy(rng.standard_normal((T, D))).to(BF16).to(DEV))
    dy = torch.from_numpy(rng.standard_normal((M, N))).to(BF16).to(DEV)
    src = torch.from_numpy(rng.permutation(M).astype(np.int32)).to(DEV)
    announce("wgrad packed large")
    got = ops.grouped_mm_wgrad_packed(dy, x, offsets(counts), E, torch.float32, src, K)
    want = ops.grouped_mm_wgrad(dy, ops.unpack_e4m3(x, src, K), offsets(counts), E, torch.float32)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


# ---------------------------------------------------------------------------
# Refusals (CPU: nothing is launched)
# ---------------------------------------------------------------------------
def _err(name, *args):
    L = importlib.import_module("torchtitan-ascend_amd._lib").load()
    assert getattr(L, name)(*args) == 1
    return L.ttamd_last_error().decode()


@pytest.mark.gpu
@pytest.mark.parametrize("C", [2048, 2056])
def test_pack_past_32_bits(ops, C):
    """More than 2^31 values: the last rows are those of a small call."""
    R, few = 1_050_001, 300
    g = torch.Generator(device=DEV).manual_seed(7)
    x = torch.randn(R, C, device=DEV, generator=g, dtype=BF16)
    announce(f"pack past 32 bits, {C} columns")
    p, q = ops.pack_e4m3(x), ops.pack_e4m3(x[R - few:])
    assert torch.equal(p.codes[R - few:], q.codes) and torch.equal(p.exponents[R - few:], q.exponents)
    del x
    small = ops.unpack_e4m3(q)
    assert torch.equal(ops.unpack_e4m3(p)[R - few:], small)
    src = torch.arange(R - 1, R - 1 - few, -1, dtype=torch.int32, device=DEV)
    assert torch.equal(ops.unpack_e4m3(p, src), small.flip(0))


@pytest.mark.gpu
@pytest.mark.parametrize("counts", [[238] * 12, [700], [3000, 0, 1, 129, 5], [64, 65, 128], [31], [4000, 1, 4000]])
@pytest.mark.parametrize("D,H", [(1024, 384), (64, 128), (1408, 512)])
def test_dgrad_packed_few_tiles(ops, counts, D, H):
    """Few tiles (shorter ones than the bf16 form's): the same bits, since a
    reduction of fewer than 24 stages of 64 is never cut and its order does not
    depend on the tiles."""
    rng = np.random.default_rng(len(counts) + D)
    M, E = sum(counts) + 3, len(counts)
    dy = torch.from_numpy(rng.standard_normal((M, D))).to(BF16).to(DEV)
    w2 = torch.from_numpy(rng.standard_normal((E, D, H)) * 0.05).to(BF16).to(DEV)
    h = ops.pack_e4m3(torch.from_numpy(rng.standard_normal((M, 2 * H))).to(BF16).to(DEV))
    announce(f"dgrad packed few tiles counts={counts} D={D} H={H}")
    n = sum(counts)
    dh, a = ops.grouped_mm_dgrad_swiglu_packed(dy, w2, h, offsets(counts), None, want_a=True)
    dh0, a0 = ops.grouped_mm_dgrad_swiglu(dy, w2, ops.unpack_e4m3(h), offsets(counts), None, want_a=True)
    assert torch.equal(dh[:n], dh0[:n]) and torch.equal(a[:n], a0[:n])


@pytest.mark.gpu
def test_dgrad_packed_past_32_bits(ops):
    """More than 2^31 codes: as from the same h in bf16."""
    D, H, last = 128, 2048, 300
    counts = [540_000, 0, last]
    M = sum(counts)
    g = torch.Generator(device=DEV).manual_seed(8)
    dy = torch.zeros(M, D, dtype=BF16, device=DEV)
    dy[M - last:] = torch.randn(last, D, device=DEV, generator=g)
    w2 = torch.randn(3, D, H, device=DEV, generator=g).to(BF16)
    h = torch.randn(last, 2 * H, device=DEV, generator=g).to(BF16)
    tail = ops.pack_e4m3(h)
    codes = torch.zeros(M, 2 * H, dtype=torch.uint8, device=DEV)
    exps = torch.full((M, 2 * H // 128), 127, dtype=torch.uint8, device=DEV)
    codes[M - last:], exps[M - last:] = tail.codes, tail.exponents
    announce("packed dgrad past 32 bits")
    dh, a = ops.grouped_mm_dgrad_swiglu_packed(dy, w2, ops.PackedRows(codes, exps), offsets(counts), want_a=True)
    hb = torch.zeros(M, 2 * H, dtype=BF16, device=DEV)
    hb[M - last:] = ops.unpack_e4m3(tail)
    want, a_want = ops.grouped_mm_dgrad_swiglu(dy, w2, hb, offsets(counts), want_a=True)
    assert want[M - last:].any()
    assert torch.equal(dh, want) and torch.equal(a, a_want)


def test_refusals():
    import ctypes

    p, odd, nan = ctypes.c_void_p(256), ctypes.c_void_p(260), float("nan")
    assert "multiple of 8" in _err("ttamd_pack_e4m3", p, 4, 12, p, p, None)
    assert "aligned" in _err("ttamd_pack_e4m3", odd, 4, 64, p, p, None)
    assert "aligned" in _err("ttamd_pack_e4m3", p, 4, 64, odd, p, None)
    assert "null" in _err("ttamd_pack_e4m3", p, 4, 64, p, None, None)
    assert "out of range" in _err("ttamd_pack_e4m3", p, -1, 64, p, p, None)
    assert "too many" in _err("ttamd_pack_e4m3", p, 1 << 28, 64, p, p, None)
    assert "too few packed rows" in _err("ttamd_unpack_e4m3", p, p, 3, 64, None, 1, None, 4, p, None)
    assert "too few packed rows" in _err("ttamd_unpack_e4m3", p, p, 0, 64, p, 1, None, 4, p, None)
    assert "src_div" in _err("ttamd_unpack_e4m3", p, p, 4, 64, p, 0, None, 4, p, None)
    assert "null" in _err("ttamd_unpack_e4m3", p, None, 4, 64, None, 1, None, 4, p, None)
    L = importlib.import_module("torchtitan-ascend_amd._lib").load()
    ws = L.ttamd_gemm_workspace_bytes(64, 2)
    dgrad = "ttamd_grouped_mm_dgrad_swiglu_packed"
    assert "hidden" in _err(dgrad, p, p, p, p, p, 64, 2, 128, 64, nan, p, p, p, ws, None)
    assert "swiglu_limit" in _err(dgrad, p, p, p, p, p, 64, 2, 128, 128, -1.0, p, p, p, ws, None)
    assert "exponents" in _err(dgrad, p, p, p, None, p, 64, 2, 128, 128, nan, p, p, p, ws, None)
    assert "workspace" in _err(dgrad, p, p, p, p, p, 64, 2, 128, 128, nan, p, p, p, ws - 1, None)
    wgrad = "ttamd_grouped_mm_wgrad_packed"
    need = L.ttamd_grouped_mm_wgrad_packed_workspace_bytes(64, 16, 2, 128, 0)
    assert need >= 16 * 128 * 2 + 64 * 4 + ws
    assert L.ttamd_grouped_mm_wgrad_packed_workspace_bytes(64, 16, 2, 128, 1) >= 64 * 128 * 2 + ws
    assert "workspace" in _err(wgrad, p, p, p, 16, p, 4, None, p, 64, 2, 128, 128, p, 1, p, need - 1, None)
    assert "multiple of 128" in _err(wgrad, p, p, p, 16, p, 4, None, p, 64, 2, 64, 128, p, 1, p, need, None)
    assert "too few packed rows" in _err(wgrad, p, p, p, 16, None, 1, None, p, 64, 2, 128, 128, p, 1, p, need, None)
    assert "src_div" in _err(wgrad, p, p, p, 16, p, 0, None, p, 64, 2, 128, 128, p, 1, p, need, None)


def test_python_refusals(ops):
    x = torch.zeros(4, 64, dtype=BF16)
    u8 = torch.zeros(4, 64, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="HIP device"):
        ops.pack_e4m3(x)
    with pytest.raises(RuntimeError, match="HIP device"):
        ops.unpack_e4m3(ops.PackedRows(u8, u8[:, :1]))
    with pytest.raises(ValueError, match="do not match"):
        ops._packed("x", ops.PackedRows(u8, u8), u8.device)
    with pytest.raises(TypeError, match="codes"):
        ops._packed("x", ops.PackedRows(x, u8[:, :1]), u8.device)


@pytest.mark.gpu
def test_dgrad_packed_few_tiles_split(ops):
    """A skewed load whose low token tiles are cut along a reduction of 32
    stages (72 tiles of 128 rows, three pieces each; an even load of as many
    experts has 100 tall ones, uncut): against 64 bits by the bound of
    test_dgrad_swiglu_packed, and the same bits every time."""
    D, H, E = 2048, 256, 100
    counts = np.zeros(E, np.int64)
    counts[[7, 50, 99]] = 3001, 2999, 3000
    M = int(counts.sum())
    gen = torch.Generator(device=DEV).manual_seed(22)
    dy = torch.randn(M, D, device=DEV, generator=gen).to(BF16)
    w2 = (torch.randn(E, D, H, device=DEV, generator=gen) * 0.05).to(BF16)
    h = ops.pack_e4m3(torch.randn(M, 2 * H, device=DEV, generator=gen).to(BF16))
    announce("dgrad packed few tiles, split")
    dh, a = ops.grouped_mm_dgrad_swiglu_packed(dy, w2, h, offsets(counts), None, want_a=True)
    torch.cuda.synchronize()
    hd = ops.unpack_e4m3(h).double().requires_grad_(True)
    act = torch.nn.functional.silu(hd[:, :H]) * hd[:, H:]
    ends = np.cumsum(counts)
    g = torch.cat([dy[ends[e] - counts[e]:ends[e]].double() @ w2[e].double() for e in (7, 50, 99)])
    (rdh,) = torch.autograd.grad(act, hd, g)
    assert rel_err_rows(to_np(dh), rdh.cpu().numpy()) < 2.0 ** -7
    assert rel_err_rows(to_np(a), act.detach().cpu().numpy()) < 2.0 ** -7
    for _ in range(3):
        dh1, a1 = ops.grouped_mm_dgrad_swiglu_packed(dy, w2, h, offsets(counts), None, want_a=True)
        assert torch.equal(dh1, dh) and torch.equal(a1, a)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, BF16])
def test_wgrad_packed_ignores_the_next_experts_special_tokens(ops, dtype):
    """A stage of 64 rows that an expert fills in part also loads the next
    experts' tokens, and behind the last row token 0: NaN and infinities there
    (NaN once packed) stay out of the gradients of experts that do not read
    them, and an expert without rows gets exact zeros."""
    rng = np.random.default_rng(21)
    counts, D, N = [30, 40, 0, 65], 256, 128
    M = sum(counts)
    x = rng.standard_normal((M, D))
    x[0, 5], x[0, 77], x[1, 9] = np.nan, np.inf, -np.inf
    src = np.roll(np.arange(M), -2)  # finite tokens ...
    src[[30, 70]] = 0, 1             # ... but the first ones of experts 1 and 3
    src[-2:] = 2, 3                  # (where tokens 0 and 1 were)
    assert src[M - 1] > 1 and (np.delete(src, [30, 70]) > 1).all()
    p = ops.pack_e4m3(torch.from_numpy(x).to(BF16).to(DEV))
    dy = torch.from_numpy(rng.standard_normal((M, N))).to(BF16).to(DEV)
    ids = torch.from_numpy(src.astype(np.int32)).to(DEV)
    announce(f"wgrad packed beside special tokens {dtype}")
    got = ops.grouped_mm_wgrad_packed(dy, p, offsets(counts), 4, dtype, ids, 1)
    want = ops.grouped_mm_wgrad(dy, ops.unpack_e4m3(p, ids, 1), offsets(counts), 4, dtype)
    torch.cuda.synchronize()
    assert bool(((got == want) | (got.isnan() & want.isnan())).all())
    nan = torch.zeros(4, N, D, dtype=torch.bool, device=DEV)
    nan[1, :, [5, 77]] = True
    nan[3, :, 9] = True
    assert torch.equal(got.isnan(), nan) and not bool(got.isinf().any())
    assert not got[2].any()


@pytest.mark.gpu
def test_every_code_and_exponent(ops):
    """Each of the 256 codes at each exponent that packing makes: exact, down to
    the least code's 2^-9 * 2^-118 = 2^-127, which bf16 and fp32 hold below
    their normal numbers.  (At e = 120 codes end at 240.)"""
    code = np.arange(256)
    mant, expo = code & 7, (code >> 3) & 15
    value = np.where(expo == 0, mant * 2.0 ** -9, (8 + mant) * np.exp2(expo - 10.0))
    value = np.where((code & 127) == 127, np.nan, value) * np.where(code & 128, -1.0, 1.0)
    bytes_ = np.arange(127 - 118, 127 + 120 + 1)
    want = value[None, :] * np.exp2(bytes_[:, None] - 127.0)
    want[-1, np.abs(value) > 240] = 0.0
    codes = np.tile(code.astype(np.uint8), (len(bytes_), 1))
    codes[-1, np.abs(value) > 240] = 0
    p = ops.PackedRows(torch.from_numpy(codes).to(DEV),
                       torch.from_numpy(np.repeat(bytes_[:, None].astype(np.uint8), 2, axis=1)).to(DEV))
    announce("every code and exponent")
    y = ops.unpack_e4m3(p).cpu().double().numpy()
    np.testing.assert_array_equal(y, want)
    # with a scale of one: the same values
    one = torch.ones(len(bytes_), device=DEV)
    np.testing.assert_array_equal(ops.unpack_e4m3(p, row_scale=one).cpu().double().numpy(), want)


@pytest.mark.gpu
def test_least_values(ops):
    """Blocks at the lowest exponent: values on, between and below the grid's
    step of 2^-127, both signs (1/2, 3/2 and 5/2 steps are ties)."""
    steps = np.array([0.0, 0.25, 0.5, 0.75, 1.0, 1.25, 1.5, 1.75, 2.0, 2.5, 3.0, 4.0, 5.5, 7.0, 8.0, 9.0, 17.0])
    x = np.concatenate([steps, -steps]) * 2.0 ** -127
    x = np.pad(x, (0, 8 - len(x) % 8))
    x = np.stack([x, np.roll(x, 5)])
    t = torch.from_numpy(x).to(BF16)
    np.testing.assert_array_equal(t.double().numpy(), x)  # bf16 holds them
    announce("least values")
    p = ops.pack_e4m3(t.to(DEV))
    e, val = define(x)
    np.testing.assert_array_equal(p.exponents.cpu().numpy(), e)
    np.testing.assert_array_equal(ops.unpack_e4m3(p).cpu().double().numpy(), val)
