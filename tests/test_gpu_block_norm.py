"""The norms around a block on the GPU against their formulas in 64 bits."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from fusion_b200 import ops
from gpu_util import finish

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _oracle(y, res, post_w, pre_w, gate, act, alpha, eps):
    d = lambda t: None if t is None else t.double().cpu().numpy()  # noqa: E731
    y, res, post_w, pre_w, gate = (d(t) for t in (y, res, post_w, pre_w, gate))
    v = y if post_w is None else y / np.sqrt((y * y).mean(1, keepdims=True) + eps) * post_w
    if gate is not None:
        v = v * {"none": lambda g: g, "sigmoid": lambda g: 1 / (1 + np.exp(-g)), "tanh": np.tanh}[act](gate)
    h = res + alpha * v
    x = None if pre_w is None else h / np.sqrt((h * h).mean(1, keepdims=True) + eps) * pre_w
    return h, x, np.abs(res) + np.abs(alpha * v)


def _check(got, want, mag, dtype, N):
    """Half a step of the type, and of fp32: the sum of N squares along a thread's share and a
    tree (N / 64 + 12 roundings, halved by the root), the gate's exponential, ten products."""
    g = got.double().cpu().numpy()
    rel = (N / 64 + 40) * 2.0 ** -24
    tol = torch.finfo(dtype).eps / 2 * (np.abs(want) + rel * mag) + rel * mag + torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    assert (np.abs(g - want) <= tol).all(), np.max(np.abs(g - want) / tol)


def _make(T, N, dtype, kind, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(T * 131 + N + seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    shape = {"none": None, "token": (T, 1), "channel": (1, N), "full": (T, N)}[kind]
    return ((3 * r(T, N)).to(dtype), r(T, N).to(dtype), (1 + 0.1 * r(N)).to(dtype),
            (1 + 0.1 * r(N)).to(dtype), r(*shape).to(dtype) if shape else None)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("kind,act", [("none", "none"), ("token", "sigmoid"), ("channel", "tanh"),
                                      ("full", "none"), ("full", "sigmoid")])
@pytest.mark.parametrize("T,N", [(1, 1), (1, 6144), (3, 7), (5, 64), (400, 96), (2, 257), (310, 1000),
                                 (301, 5003), (299, 6144), (2, 16384)])
def test_matches_formula(dtype, kind, act, T, N):
    dt = DTYPES[dtype]
    y, res, post_w, pre_w, gate = _make(T, N, dt, kind)
    h, x = torch.empty_like(y), torch.empty_like(y)
    ops.norm_gate_residual(y, res, h, x, post_w=post_w, pre_w=pre_w, gate=gate, gate_act=act, alpha=0.37, eps=1e-5)
    finish()
    wh, wx, mag = _oracle(y, res, post_w, pre_w, gate, act, np.float32(0.37), np.float32(1e-5))
    _check(h, wh, mag, dt, N)
    _check(x, wx, np.abs(wx) + mag * np.abs(pre_w.double().cpu().numpy()) /
           np.sqrt((wh * wh).mean(1, keepdims=True) + 1e-5), dt, N)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("kind,act", [("none", "none"), ("token", "tanh"), ("channel", "tanh"),
                                      ("full", "sigmoid")])
@pytest.mark.parametrize("T,N", [(600, 6144), (593, 1536), (1200, 2048), (601, 5003), (900, 2049), (592, 1035),
                                 (700, 3071)])
def test_many_rows(dtype, kind, act, T, N):
    """Batches that go through the ring of rows, whole 16-byte lines and odd widths."""
    dt = DTYPES[dtype]
    y, res, post_w, pre_w, gate = _make(T, N, dt, kind)
    h, x = torch.empty_like(y), torch.empty_like(y)
    ops.norm_gate_residual(y, res, h, x, post_w=post_w, pre_w=pre_w, gate=gate, gate_act=act, alpha=0.37, eps=1e-5)
    h1 = torch.empty_like(y)
    ops.norm_gate_residual(y, res, h1, gate=gate, gate_act=act, alpha=0.37)
    r2, y2 = res.clone(), y.clone()  # in place
    ops.norm_gate_residual(y2, r2, r2, y2, post_w=post_w, pre_w=pre_w, gate=gate, gate_act=act, alpha=0.37, eps=1e-5)
    finish()
    wh, wx, mag = _oracle(y, res, post_w, pre_w, gate, act, np.float32(0.37), np.float32(1e-5))
    _check(h, wh, mag, dt, N)
    _check(x, wx, np.abs(wx) + mag * np.abs(pre_w.double().cpu().numpy()) /
           np.sqrt((wh * wh).mean(1, keepdims=True) + 1e-5), dt, N)
    wh1, _, mag1 = _oracle(y, res, None, None, gate, act, np.float32(0.37), np.float32(1e-5))
    _check(h1, wh1, mag1, dt, N)
    assert torch.equal(r2, h) and torch.equal(y2, x)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("kind,act", [("none", "none"), ("channel", "tanh"), ("full", "sigmoid")])
@pytest.mark.parametrize("T,N", [(2071, 521), (2072, 505), (2072, 512), (3001, 1021), (2503, 259), (2200, 253)])
def test_many_narrow_rows(dtype, kind, act, T, N):
    test_many_rows(dtype, kind, act, T, N)


@pytest.mark.parametrize("ld,first", [(523, 0), (524, 1), (525, 2), (526, 3), (527, 4), (528, 5), (529, 6), (530, 7)])
@pytest.mark.parametrize("N", [515, 521, 523])
def test_every_end_of_a_row(N, ld, first):
    """Rows that start and end at every place of a 16-byte line; what lies beside them stays."""
    T = 2080
    y0, res0, post_w, pre_w, _ = _make(T, N, torch.float16, "none")
    bufs = [torch.full((first + T * ld,), 5.0, dtype=torch.float16, device="cuda") for _ in range(4)]
    y, res, h, x = (b[first:].as_strided((T, N), (ld, 1)) for b in bufs)
    y.copy_(y0), res.copy_(res0)
    ops.norm_gate_residual(y, res, h, x, post_w=post_w, pre_w=pre_w)
    finish()
    wh, wx, mag = _oracle(y0, res0, post_w, pre_w, None, "none", 1.0, np.float32(1e-5))
    _check(h, wh, mag, torch.float16, N)
    _check(x, wx, np.abs(wx) + mag, torch.float16, N)
    for b, got in ((bufs[2], h), (bufs[3], x)):
        gone = b.clone()
        gone[first:].as_strided((T, N), (ld, 1)).fill_(5.0)
        assert bool((gone == 5.0).all())


def test_many_rows_apart():
    """Strided rows through the ring: what lies between them is neither read nor written."""
    T, N, ld = 640, 1501, 1533
    for off in (0, 3, 8):
        y0, res0, post_w, pre_w, gate0 = _make(T, N, torch.bfloat16, "full")
        bufs = [torch.full((off + (T - 1) * ld + N,), float("nan"), dtype=torch.bfloat16, device="cuda")
                for _ in range(5)]
        y, res, h, x, gate = (b[off:].as_strided((T, N), (ld, 1)) for b in bufs)
        y.copy_(y0), res.copy_(res0), gate.copy_(gate0)
        h.fill_(7.0), x.fill_(7.0)
        ops.norm_gate_residual(y, res, h, x, post_w=post_w, pre_w=pre_w, gate=gate, gate_act="sigmoid")
        finish()
        wh, wx, mag = _oracle(y0, res0, post_w, pre_w, gate0, "sigmoid", 1.0, np.float32(1e-5))
        _check(h, wh, mag, torch.bfloat16, N)
        _check(x, wx, np.abs(wx) + mag, torch.bfloat16, N)
        for b in (bufs[2], bufs[3]):
            assert int(torch.isnan(b).sum()) == b.numel() - T * N


def test_widest_rows():
    for dt, N in ((torch.bfloat16, 32768), (torch.float32, 16384)):
        y, res, post_w, pre_w, _ = _make(2, N, dt, "none")
        h, x = torch.empty_like(y), torch.empty_like(y)
        ops.norm_gate_residual(y, res, h, x, post_w=post_w, pre_w=pre_w)
        finish()
        wh, wx, mag = _oracle(y, res, post_w, pre_w, None, "none", 1.0, np.float32(1e-5))
        _check(h, wh, mag, dt, N)
        _check(x, wx, np.abs(wx) + mag, dt, N)
        wide = torch.zeros(1, 2 * N + 8, dtype=dt, device="cuda")
        with pytest.raises(RuntimeError, match="too wide"):
            ops.norm_gate_residual(wide, wide, wide)


@pytest.mark.parametrize("post,pre", [(False, False), (False, True), (True, False)])
def test_optional_norms(post, pre):
    y, res, post_w, pre_w, gate = _make(17, 320, torch.bfloat16, "token")
    h = torch.empty_like(y)
    x = torch.empty_like(y) if pre else None
    ops.norm_gate_residual(y, res, h, x, post_w=post_w if post else None, pre_w=pre_w if pre else None, alpha=0.22)
    finish()
    wh, wx, mag = _oracle(y, res, post_w if post else None, pre_w if pre else None, None, "none",
                          np.float32(0.22), np.float32(1e-5))
    _check(h, wh, mag, torch.bfloat16, 320)
    if pre:
        _check(x, wx, np.abs(wx) + mag, torch.bfloat16, 320)


@pytest.mark.parametrize("off,ld", [((0, 0, 0, 0), 320), ((1, 1, 1, 1), 301), ((3, 3, 3, 3), 304),
                                    ((0, 1, 2, 3), 307), ((8, 8, 0, 0), 312)])
def test_strides_and_alignments(off, ld):
    """Rows anywhere, alike or not; what lies between rows stays."""
    T, N = 9, 299
    y0, res0, post_w, pre_w, gate0 = _make(T, N, torch.bfloat16, "full")
    bufs = [torch.full((T * ld + 16,), 5.0, dtype=torch.bfloat16, device="cuda") for _ in range(5)]
    y, res, h, x, gate = (b[o:].as_strided((T, N), (ld, 1)) for b, o in zip(bufs, off + (off[0],)))
    y.copy_(y0), res.copy_(res0), gate.copy_(gate0)
    ops.norm_gate_residual(y, res, h, x, post_w=post_w, pre_w=pre_w, gate=gate, gate_act="sigmoid")
    finish()
    wh, wx, mag = _oracle(y0, res0, post_w, pre_w, gate0, "sigmoid", 1.0, np.float32(1e-5))
    _check(h, wh, mag, torch.bfloat16, N)
    _check(x, wx, np.abs(wx) + mag, torch.bfloat16, N)
    for b, o in ((bufs[2], off[2]), (bufs[3], off[3])):
        hole = torch.ones(b.numel(), dtype=torch.bool, device="cuda")
        hole[o:].as_strided((T, N), (ld, 1)).fill_(False)
        assert (b[hole] == 5.0).all()


@pytest.mark.parametrize("T", [7, 700])
@pytest.mark.parametrize("off", [1, 4])
def test_weights_anywhere(T, off):
    """Norm weights and a channel gate that do not start on 16 bytes."""
    for N in (1200, 1203):
        y, res, post_w, pre_w, gate = _make(T, N, torch.bfloat16, "channel")
        post_w, pre_w, gate = (torch.cat([t.reshape(-1)[:1].expand(off), t.reshape(-1)])[off:] for t in (post_w, pre_w, gate))
        h, x = torch.empty_like(y), torch.empty_like(y)
        ops.norm_gate_residual(y, res, h, x, post_w=post_w, pre_w=pre_w, gate=gate, gate_act="sigmoid")
        finish()
        wh, wx, mag = _oracle(y, res, post_w, pre_w, gate, "sigmoid", 1.0, np.float32(1e-5))
        _check(h, wh, mag, torch.bfloat16, N)
        _check(x, wx, np.abs(wx) + mag, torch.bfloat16, N)


def test_in_place():
    """h over res, h over y, x over y: the row is read before it is written."""
    for N in (512, 509):
        y, res, post_w, pre_w, _ = _make(33, N, torch.bfloat16, "none")
        h, x = torch.empty_like(y), torch.empty_like(y)
        ops.norm_gate_residual(y, res, h, x, post_w=post_w, pre_w=pre_w)
        y1, r1 = y.clone(), res.clone()
        ops.norm_gate_residual(y1, r1, r1, y1, post_w=post_w, pre_w=pre_w)
        y2, x2 = y.clone(), torch.empty_like(y)
        ops.norm_gate_residual(y2, res, y2, x2, post_w=post_w, pre_w=pre_w)
        finish()
        assert torch.equal(r1, h) and torch.equal(y1, x) and torch.equal(y2, h) and torch.equal(x2, x)


def test_infinities_stay_in_their_rows():
    y, res, post_w, pre_w, _ = _make(6, 96, torch.bfloat16, "none")
    y[1, 3] = float("inf")
    res[4, 90] = float("nan")
    h, x = torch.empty_like(y), torch.empty_like(y)
    ops.norm_gate_residual(y, res, h, x, post_w=post_w, pre_w=pre_w)
    finish()
    ok = torch.isfinite(x).all(1).tolist()
    assert ok == [True, False, True, True, False, True]


def test_graph_on_another_stream_and_empty_batch():
    y, res, post_w, pre_w, _ = _make(64, 1024, torch.bfloat16, "none")
    h, x = torch.empty_like(y), torch.empty_like(y)
    ops.norm_gate_residual(y, res, h, x, post_w=post_w, pre_w=pre_w)
    h2, x2 = torch.zeros_like(y), torch.zeros_like(y)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.norm_gate_residual(y, res, h2, x2, post_w=post_w, pre_w=pre_w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        g.replay()
    finish()
    assert torch.equal(h, h2) and torch.equal(x, x2)
    ops.norm_gate_residual(y[:0], res[:0], h[:0], x[:0], post_w=post_w, pre_w=pre_w)
    finish()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("T,N", [(8000, 1536), (4001, 6144), (3001, 5003), (9001, 515), (6000, 512)])
def test_many_rows_without_the_next_norm(dtype, T, N):
    """Many rows of a CTA one after another, one sum each: the sums do not run into one another. The
    same arithmetic with the next norm gives the same h, bit for bit."""
    dt = DTYPES[dtype]
    y, res, post_w, pre_w, gate = _make(T, N, dt, "token")
    y *= torch.exp(torch.randn(T, 1, device="cuda")).to(dt)  # every row a sum of its own
    want, x = torch.empty_like(y), torch.empty_like(y)
    ops.norm_gate_residual(y, res, want, x, post_w=post_w, pre_w=pre_w, gate=gate, gate_act="sigmoid", alpha=0.37)
    for _ in range(5):
        h = torch.full_like(y, 9.0)
        ops.norm_gate_residual(y, res, h, post_w=post_w, gate=gate, gate_act="sigmoid", alpha=0.37)
        assert torch.equal(h, want)
    finish()
    wh, _, mag = _oracle(y, res, post_w, None, gate, "sigmoid", np.float32(0.37), np.float32(1e-5))
    _check(h, wh, mag, dt, N)
