"""Microscaled 4-bit floating point on the GPU against 64-bit oracles: every code and scale
byte bit for bit, products within the rounding of their sums."""

from __future__ import annotations

import pathlib
import subprocess
import sys
import threading

import numpy as np
import pytest
import torch

import fp4_oracle as Q
from fusion_b200 import fp4, ops
from gpu_util import finish

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _quantize(x, fmt, tile, g=None, rows=None, **kw):
    rows = x.shape[0] if rows is None else rows
    K = x.shape[1]
    q = torch.full((rows, K // 2), 0xEE, dtype=torch.uint8, device="cuda")
    sf = torch.full((ops.fp4_scale_bytes(rows, K, fmt, tile),), 0xEE, dtype=torch.uint8, device="cuda")
    ops.fp4_quantize(x, q, sf, fmt, tile=tile, gscale=g, **kw)
    finish()
    return q, sf


def _scales(sf, fmt, rows, K, tile):
    s = sf.cpu().numpy()
    if tile == 0:
        return s.reshape(rows, -1)
    return s[Q.scale_positions(fmt, rows, K, tile)]


def _check(x, fmt, tile, g=None, per_row=1.0):
    R, K = x.shape
    q, sf = _quantize(x, fmt, tile, g)
    code, byte = Q.quantize(x.double().cpu().numpy(), fmt, per_row)
    np.testing.assert_array_equal(_scales(sf, fmt, R, K, tile), byte)
    got = Q.unpack(q.cpu().numpy())
    # the sign of a zero carries no value
    np.testing.assert_array_equal(np.where(got == 8, 0, got), np.where(code == 8, 0, code))
    return q, sf, code, byte


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,K,tile", [(1, 32, 0), (3, 64, 16), (33, 96, 32), (129, 288, 64),
                                         (200, 544, 128), (300, 2080, 256), (64, 6144, 128)])
def test_quantize_matches_definition(fmt, dtype, rows, K, tile):
    gen = torch.Generator(device="cuda").manual_seed(rows * K)
    x = torch.randn(rows, K, device="cuda", generator=gen) * torch.exp(
        3 * torch.randn(rows, 1, device="cuda", generator=gen))
    x = x.to(DTYPES[dtype])
    g = torch.tensor([0.0123], device="cuda") if fmt == "nv" else None
    q, sf, code, byte = _check(x, fmt, tile, g, g.item() if g is not None else 1.0)
    # and back: one rounding of the factor, one of the type
    out = torch.empty_like(x)
    ops.fp4_dequantize(q, sf, out, fmt, tile=tile, gscale=g)
    finish()
    want = Q.values(code, byte, fmt, float(g.item()) if g is not None else 1.0)
    eps = torch.finfo(x.dtype).eps / 2 + 2.0 ** -24
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    top = float(torch.finfo(x.dtype).max)
    got = out.double().cpu().numpy()
    fits = np.abs(want) < top
    assert (np.abs(got - want)[fits] <= eps * np.abs(want[fits]) + tiny).all()


@pytest.mark.parametrize("fmt", ["mx", "nv"])
def test_quantize_special_values(fmt):
    K = 64
    x = torch.zeros(12, K)
    x[1] = -0.0
    x[2, 5] = float("inf")
    x[3, 40] = float("nan")
    x[4, 63] = -float("inf")
    x[5] = 1e-45  # subnormal
    x[6, ::3] = 3e38
    x[7] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 8)  # ties
    x[8] = -x[7]
    x[9] = x[7] * 2.0 ** -130
    x[10, 3] = 1e-38
    x[11] = torch.linspace(-6, 6, K)
    _check(x.cuda(), fmt, 16)
    _check(x.cuda(), fmt, 0)


def test_quantize_nv_next_to_the_borders():
    """Values that fp32 division puts on the wrong side of a rounding border: next neighbours
    of border * scale * g, and amax next to the border between two e4m3 scales."""
    rng = np.random.default_rng(5)
    rows, K = 512, 32
    g = np.float32(rng.uniform(0.5, 2.0, rows))
    x = np.zeros((rows, K), dtype=np.float32)
    borders = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    for r in range(rows):
        s = Q.E4M3[rng.integers(8, 126)] * np.float64(g[r])
        x[r, 0] = 6.0 * s  # keeps the block's scale at s
        b = np.float32(np.tile(borders, 3)[:15] * s)
        x[r, 1:16] = np.nextafter(b, np.float32(rng.choice([-1e30, 1e30])))
        i = rng.integers(8, 125)
        m = 0.5 * (Q.E4M3[i] + Q.E4M3[i + 1]) * 6.0 * np.float64(g[r])
        x[r, 16] = np.nextafter(np.float32(m), np.float32(rng.choice([0.0, 1e30])))
    _check(torch.from_numpy(x).cuda(), "nv", 128, torch.from_numpy(g).cuda(), g.astype(np.float64))


@pytest.mark.parametrize("g", [1e-38, 1e-20, 3e37])
def test_quantize_nv_extreme_factors(g):
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(20, 96, device="cuda", generator=gen)
    gt = torch.tensor([g], device="cuda")
    _check(x, "nv", 32, gt, float(gt.item()))


@pytest.mark.parametrize("offset,ld", [(0, 100), (1, 97), (3, 112), (16, 128)])
def test_quantize_strided_rows(offset, ld):
    buf = torch.randn(40, ld + 16, device="cuda").to(torch.bfloat16)
    x = buf.view(-1)[offset:offset + 39 * ld + 64].as_strided((39, 64), (ld, 1))
    _check(x, "mx", 64)
    _check(x, "nv", 64)


@pytest.mark.parametrize("fmt", ["mx", "nv"])
def test_quantize_gathered_rows_and_pads(fmt):
    """Row p is x[ids[p] // 3]; pads, ids out of range and rows from ntp on keep their bytes."""
    K, T, k = 288, 5, 3
    x = torch.randn(T, K, device="cuda").to(torch.bfloat16)
    ids = torch.tensor([4, 0, 14, 15, 15, -1, 7, 1, 99, 2, 3, 4], dtype=torch.int32, device="cuda")
    ntp = torch.tensor([9], dtype=torch.int32, device="cuda")
    q, sf = _quantize(x, fmt, 16, rows=12, ids=ids, id_div=k, id_limit=T * k, ntp=ntp)
    code, byte = Q.quantize(x.double().cpu().numpy(), fmt)
    s = _scales(sf, fmt, 12, K, 16)
    for p, i in enumerate(ids.tolist()):
        if p < 9 and 0 <= i < T * k:
            np.testing.assert_array_equal(q[p].cpu().numpy(), Q.pack(code[i // k]))
            np.testing.assert_array_equal(s[p], byte[i // k])
        else:
            assert (q[p] == 0xEE).all() and (s[p] == 0xEE).all()


def _stack(E, N, K, fmt, seed):
    w = torch.randn(E, N, K, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))
    q, s, g = fp4.quantize_weight((w * 0.05).to(torch.bfloat16), fmt)
    gn = g.double().cpu().numpy()[:, None, None] if g is not None else 1.0
    val = Q.values(Q.unpack(q.cpu().numpy()), s.cpu().numpy(), fmt, gn)
    return q, s, g, val


def _reference(x, w, topi, swiglu):
    """Rows [T*k, cols] in 64 bits and the bound of |y| from the sums' rounding.

    The tensor core adds exact products in fp32, one rounding (toward zero at worst, 2^-23)
    for each partial sum of at least 16 terms, the scale and factor two more: (K/16 + 4) 2^-23
    of the sum of magnitudes."""
    T, k = topi.shape
    K = x.shape[1]
    y = np.stack([w[topi[t, j]] @ x[t] for t in range(T) for j in range(k)])
    mag = np.stack([np.abs(w[topi[t, j]]) @ np.abs(x[t]) for t in range(T) for j in range(k)])
    err = (K / 16 + 4) * 2.0 ** -23 * mag
    if swiglu:
        a, b = np.split(y, 2, -1)
        da, db = np.split(err, 2, -1)
        with np.errstate(over="ignore"):
            silu = a / (1 + np.exp(-a))
        y = silu * b
        # |silu'| <= 1.1; the fast exponential and division are within 2^-20
        err = 1.1 * da * np.abs(b) + np.abs(silu) * db + 1.1 * da * db + 2.0 ** -20 * np.abs(y)
    return y, err


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("T,k,E,N,K,bn", [
    (1, 1, 1, 16, 32, 16), (1, 2, 4, 128, 256, 16), (9, 2, 5, 144, 288, 16), (40, 2, 4, 272, 544, 32),
    (70, 3, 5, 400, 96, 64), (150, 2, 3, 208, 800, 128), (300, 2, 3, 256, 1024, 256),
    (37, 4, 4, 528, 2080, 256), (500, 1, 2, 64, 64, 16)])
def test_expert_product(fmt, swiglu, T, k, E, N, K, bn):
    rng = np.random.default_rng(T * N + K)
    topi = np.stack([rng.choice(E, k, replace=False) for _ in range(T)])
    x = torch.randn(T, K, device="cuda", generator=torch.Generator(device="cuda").manual_seed(T)).to(torch.bfloat16)
    q, s, g, w = _stack(E, N, K, fmt, 1)
    xg = torch.tensor([0.0021], device="cuda") if fmt == "nv" else None
    proj = fp4.ExpertGemmFP4(q, s, fmt, gscale=g, x_gscale=xg, gate_up=swiglu)
    ids, eids, total = Q.layout(topi, E, bn, extra=2)
    dev = [torch.from_numpy(v).cuda() for v in (ids, eids, np.array([total], dtype=np.int32))]
    xf = float(xg.item()) if xg is not None else 1.0
    xv = Q.values(*Q.quantize(x.double().cpu().numpy(), fmt, xf), fmt, xf)
    want, err = _reference(xv, w, topi, swiglu)
    scale = torch.rand(T * k + 3, device="cuda")
    for dtype, rs in ((torch.bfloat16, None), (torch.float32, scale)):
        out = torch.full((T * k + 3, proj.cols + 8), 77.0, dtype=dtype, device="cuda")[:, :proj.cols]
        proj(x, out, *dev, bn, topk=k, row_scale=rs)
        finish()
        got = out.double().cpu().numpy()
        assert (got[T * k:] == 77.0).all()  # rows behind the last pair
        f = rs[:T * k].double().cpu().numpy()[:, None] if rs is not None else 1.0
        step = torch.finfo(dtype).eps / 2 + 2.0 ** -23
        assert (np.abs(got[:T * k] - want * f) <= err * f + step * np.abs(want * f) + 1e-30).all()
    # dispatch order, rows already there: pads and junk blocks stay as they were
    xs = torch.zeros(len(ids), K, dtype=torch.bfloat16, device="cuda")
    live = ids < T * k
    live[total:] = False
    at = torch.from_numpy(np.flatnonzero(live)).cuda()
    xs[at] = x[torch.from_numpy(ids[live].astype(np.int64)).cuda() // k]
    out = torch.full((len(ids), proj.cols), 77.0, dtype=torch.bfloat16, device="cuda")
    pairs_out = torch.empty(T * k, proj.cols, dtype=torch.bfloat16, device="cuda")
    proj(xs, pairs_out, *dev, bn, gather=False)
    proj(x, out, *dev, bn, topk=k, scatter=False)
    finish()
    got = out.double().cpu().numpy()
    assert (got[~live] == 77.0).all()
    assert torch.equal(out[at], pairs_out[torch.from_numpy(ids[live].astype(np.int64)).cuda()])
    d = got[live] - want[ids[live]]
    assert (np.abs(d) <= err[ids[live]] + (2.0 ** -8 + 2.0 ** -23) * np.abs(want[ids[live]]) + 1e-30).all()


def test_expert_product_nan_rows_stay_apart():
    """A NaN in one token spoils that token's rows and no other."""
    x = torch.randn(6, 64, device="cuda").to(torch.bfloat16)
    x[2, 7] = float("nan")
    x[4, 40] = float("inf")
    q, s, g, _ = _stack(2, 32, 64, "nv", 3)
    ids, eids, total = Q.layout(np.array([[0], [0], [0], [1], [1], [0]]), 2, 16)
    dev = [torch.from_numpy(v).cuda() for v in (ids, eids, np.array([total], dtype=np.int32))]
    out = torch.empty(6, 32, dtype=torch.bfloat16, device="cuda")
    fp4.ExpertGemmFP4(q, s, "nv", gscale=g)(x, out, *dev, 16)
    finish()
    bad = torch.isnan(out).all(1).tolist()
    assert bad == [False, False, True, False, True, False]
    assert torch.isfinite(out[[0, 1, 3, 5]]).all()


def test_expert_product_bad_expert_is_reported():
    x = torch.randn(2, 64, device="cuda").to(torch.bfloat16)
    q, s, g, _ = _stack(2, 32, 64, "mx", 3)
    ids = torch.full((32,), 2, dtype=torch.int32, device="cuda")
    ids[0], ids[16] = 0, 1
    eids = torch.tensor([0, 5], dtype=torch.int32, device="cuda")
    ntp = torch.tensor([32], dtype=torch.int32, device="cuda")
    out = torch.full((2, 32), 5.0, dtype=torch.bfloat16, device="cuda")
    fp4.ExpertGemmFP4(q, s, "mx")(x, out, ids, eids, ntp, 16)
    torch.cuda.synchronize()
    assert ops.read_status() == ops.ERR_BAD_EXPERT
    assert (out[1] == 5.0).all() and not (out[0] == 5.0).all()


def test_expert_product_streams_and_graphs():
    """Two captured graphs and eager calls on two streams, all at once, share nothing."""
    E, N, K, T, k, bn = 4, 256, 512, 24, 2, 16
    q, s, g, _ = _stack(E, N, K, "nv", 7)
    proj = fp4.ExpertGemmFP4(q, s, "nv", gscale=g, gate_up=True)
    rng = np.random.default_rng(1)
    topi = np.stack([rng.choice(E, k, replace=False) for _ in range(T)])
    ids, eids, total = Q.layout(topi, E, bn)
    dev = [torch.from_numpy(v).cuda() for v in (ids, eids, np.array([total], dtype=np.int32))]
    xs = [torch.randn(T, K, device="cuda").to(torch.bfloat16) for _ in range(4)]
    want = [proj(x, torch.empty(T * k, N // 2, dtype=torch.bfloat16, device="cuda"), *dev, bn, topk=k)
            for x in xs]
    outs = [torch.zeros_like(want[0]) for _ in xs]
    graphs = []
    for i in (0, 1):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            proj(xs[i], outs[i], *dev, bn, topk=k)
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                if i < 2:
                    graphs[i].replay()
                else:
                    proj(xs[i], outs[i], *dev, bn, topk=k)
    finish()
    for a, b in zip(outs, want):
        assert torch.equal(a, b)


def test_empty_batch():
    q, s, g, _ = _stack(2, 32, 64, "mx", 3)
    e = torch.empty(0, dtype=torch.int32, device="cuda")
    ntp = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.empty(0, 32, dtype=torch.bfloat16, device="cuda")
    fp4.ExpertGemmFP4(q, s, "mx")(torch.empty(0, 64, dtype=torch.bfloat16, device="cuda"), out, e, e, ntp, 16)
    ops.fp4_quantize(torch.empty(0, 64, device="cuda"), torch.empty(0, 32, dtype=torch.uint8, device="cuda"),
                     torch.empty(0, dtype=torch.uint8, device="cuda"), "nv")
    finish()


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("T,N,K", [(1, 48, 96), (17, 256, 256), (100, 400, 544), (500, 144, 320)])
def test_dense_product(fmt, T, N, K):
    """One weight, every row: no layout."""
    q, s, g, w = _stack(1, N, K, fmt, 4)
    x = torch.randn(T, K, device="cuda").to(torch.float16)
    out = torch.full((T + 1, N), 5.0, dtype=torch.float32, device="cuda")
    fp4.ExpertGemmFP4(q, s, fmt, gscale=g)(x, out)
    finish()
    xv = Q.values(*Q.quantize(x.double().cpu().numpy(), fmt), fmt)
    ref, mag = xv @ w[0].T, np.abs(xv) @ np.abs(w[0]).T
    got = out.double().cpu().numpy()
    assert (got[T] == 5.0).all()
    assert (np.abs(got[:T] - ref) <= (K / 16 + 8) * 2.0 ** -23 * mag + 1e-30).all()


@pytest.mark.parametrize("fmt", ["mx", "nv"])
def test_large_batch_quantises_tokens_once(fmt):
    """Enough pairs that tokens are quantised once and written to their pairs' rows: the same bits as
    one pass over the dispatch order gives. Holes, pads and junk behind the layout included."""
    T, k, E, N, K, bn = 900, 6, 4, 32, 1024, 256
    rng = np.random.default_rng(3)
    topi = rng.integers(0, E, (T, k))
    ids, eids, total = Q.layout(topi, E, bn, extra=1)
    hole = ids == 77  # a pair that is not placed
    ids[hole] = T * k
    dev = [torch.from_numpy(v).cuda() for v in (ids, eids, np.array([total], dtype=np.int32))]
    x = torch.randn(T, K, device="cuda").to(torch.bfloat16)
    q, s, g, _ = _stack(E, N, K, fmt, 8)
    proj = fp4.ExpertGemmFP4(q, s, fmt, gscale=g)
    out = torch.full((T * k, N), 3.0, dtype=torch.bfloat16, device="cuda")
    proj(x, out, *dev, bn, topk=k)
    # rows already in dispatch order take the other way
    live = (ids < T * k) & (np.arange(len(ids)) < total)
    xs = torch.zeros(len(ids), K, dtype=torch.bfloat16, device="cuda")
    at = torch.from_numpy(np.flatnonzero(live)).cuda()
    xs[at] = x[torch.from_numpy(ids[live].astype(np.int64)).cuda() // k]
    want = torch.full((T * k, N), 3.0, dtype=torch.bfloat16, device="cuda")
    proj(xs, want, *dev, bn, gather=False)
    finish()
    assert torch.equal(out, want) and (out[77] == 3.0).all()


def test_expert_product_refuses_and_leaves():
    """No slots, negative pairs, an empty total; an empty batch leaves a longer output as it was."""
    E, N, K, bn = 2, 64, 64, 16
    q, s, g, _ = _stack(E, N, K, "nv", 3)
    proj = fp4.ExpertGemmFP4(q, s, "nv", gscale=g)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    lay = (torch.zeros(16, dtype=torch.int32, device="cuda"), i32(0), i32(16))
    x = torch.zeros(4, K, dtype=torch.bfloat16, device="cuda")
    out = torch.full((16, N), 7.0, dtype=torch.bfloat16, device="cuda")
    for bad in (dict(topk=0), dict(topk=-1), dict(gather=False, pairs=-1)):
        with pytest.raises(ValueError, match="not possible"):
            proj(x, out, *lay, bn, **bad)
    with pytest.raises(ValueError, match="padded total"):
        proj(x, out, lay[0], lay[1], lay[2][:0], bn, topk=4)
    proj(x[:0], out, *lay, bn, topk=4)
    ops.fp4_quantize(x, torch.zeros(16, K // 2, dtype=torch.uint8, device="cuda"),
                     torch.zeros(ops.fp4_scale_bytes(16, K, "nv", bn), dtype=torch.uint8, device="cuda"),
                     "nv", tile=bn, ids=lay[0], id_limit=2 ** 40)
    finish()
    assert bool((out == 7.0).all())


@pytest.mark.parametrize("T,bn", [(3, 16), (400, 128)])
def test_two_threads_on_one_stream(T, bn):
    """Threads share the default stream: their calls' launches fall between one another, and each
    call's packed rows stay its own."""
    E, N, K, k = 4, 256, 1024, 2
    q, s, g, _ = _stack(E, N, K, "nv", 7)
    proj = fp4.ExpertGemmFP4(q, s, "nv", gscale=g, gate_up=True)
    rng = np.random.default_rng(T)
    topi = np.stack([rng.choice(E, k, replace=False) for _ in range(T)])
    ids, eids, total = Q.layout(topi, E, bn)
    dev = [torch.from_numpy(v).cuda() for v in (ids, eids, np.array([total], dtype=np.int32))]
    xs = [torch.randn(T, K, device="cuda").to(torch.bfloat16) for _ in range(3)]
    new = lambda: torch.empty(T * k, N // 2, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    want = [proj(x, new(), *dev, bn, topk=k) for x in xs]
    outs = [[new() for _ in range(60)] for _ in xs]
    finish()
    start = threading.Barrier(len(xs))

    def calls(x, mine):
        start.wait()
        for out in mine:
            proj(x, out, *dev, bn, topk=k)

    threads = [threading.Thread(target=calls, args=a) for a in zip(xs, outs)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    finish()
    for mine, w in zip(outs, want):
        assert all(torch.equal(out, w) for out in mine)


@pytest.mark.parametrize("dtype,g", [("bf16", 2e-30), ("fp32", 1e-28), ("bf16", 0.04), ("fp16", 2e-30)])
def test_quantize_nv_values_past_the_factor(dtype, g):
    """Finite values whose quotient by the factor is past e4m3's largest, and past fp32's: the scale
    is 448, the codes saturate."""
    dt = DTYPES[dtype]
    gen = torch.Generator(device="cuda").manual_seed(7)
    x = torch.randn(24, 96, device="cuda", generator=gen)
    x[::3] *= torch.finfo(dt).max / 8
    x[1::3, ::5] *= torch.finfo(dt).max / 8
    gt = torch.tensor([g], device="cuda")
    _check(x.to(dt), "nv", 32, gt, float(gt.item()))


def test_first_call_captured():
    """A process whose first call is recorded in a graph: replays do not clear what other calls
    reported (the status word belongs to the process, not to the graph)."""
    code = """
import torch
from fusion_b200 import fp4, ops
q, s = torch.zeros(2, 32, 32, dtype=torch.uint8, device="cuda"), torch.zeros(2, 32, 4, dtype=torch.uint8, device="cuda")
i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
x, w, i = torch.randn(4, 16, device="cuda"), torch.empty(4, 2, device="cuda"), torch.empty(4, 2, dtype=torch.int32, device="cuda")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    ops.route_topk(x, w, i)
graph.replay()
ops.check_status()
assert (w.sum(1) - 1).abs().max() < 1e-6
ids = torch.full((16,), 1, dtype=torch.int32, device="cuda")
ids[0] = 0
out = torch.zeros(1, 32, dtype=torch.bfloat16, device="cuda")
fp4.ExpertGemmFP4(q, s, "nv")(torch.zeros(1, 64, dtype=torch.bfloat16, device="cuda"), out, ids, i32(7), i32(16), 16)
graph.replay()
torch.cuda.synchronize()
assert ops.read_status() == ops.ERR_BAD_EXPERT
"""
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=200,
                         cwd=pathlib.Path(__file__).parent.parent)
    assert run.returncode == 0, run.stderr[-2000:]
