"""Microscaled 4-bit floating point without a GPU: sizes, refusals, and the oracle itself."""

from __future__ import annotations

import ctypes
import weakref

import numpy as np
import pytest
import torch

import fp4_oracle as Q
from fusion_b200 import _lib as L
from fusion_b200 import fp4, ops

P = 0x10000  # a 256-byte aligned address that host checks never read


def test_oracle_grids():
    assert list(Q.E2M1) == [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    assert Q.E4M3[126] == 448 and Q.E4M3[1] == 2.0 ** -9
    # ties to the even code, saturation at the top
    assert list(Q.nearest(Q.E2M1, np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 9.0]))) == [0, 2, 2, 4, 4, 6, 6, 7]


@pytest.mark.parametrize("fmt,n", [("mx", 32), ("nv", 16)])
def test_scale_bytes(fmt, n):
    assert ops.fp4_scale_bytes(5, 96, fmt, 0) == 5 * 96 // n
    for tile in (16, 32, 64, 128, 256):
        for rows in (1, 16, 257):
            for K in (32, 256, 6144):
                pos = Q.scale_positions(fmt, rows, K, tile)
                size = ops.fp4_scale_bytes(rows, K, fmt, tile)
                assert size > pos.max() and len(np.unique(pos)) == pos.size
                assert size == L.lib().fus_fp4_scale_bytes(ops.FP4_FORMATS[fmt], rows, K, tile)
    with pytest.raises(ValueError):
        ops.fp4_scale_bytes(4, 40, fmt)
    with pytest.raises(ValueError):
        ops.fp4_scale_bytes(4, 64, fmt, tile=48)


def _refused(rc, text):
    assert rc in (-1, -3) and text in L.last_error(), L.last_error()


def test_quantize_refusals():
    def call(x=P, dtype=0, ldx=64, x_rows=4, K=64, fmt=1, g=None, per=0, ids=None, div=1, limit=0,
             rows=4, tile=16, q=P, ldq=32, sf=P):
        return L.lib().fus_fp4_quantize(x, dtype, ldx, x_rows, K, fmt, g, per, ids, div, limit, None,
                                        rows, tile, q, ldq, sf, None, None)

    assert call(rows=0) == 0
    _refused(call(K=40), "multiple of 32")
    _refused(call(K=0), "multiple of 32")
    _refused(call(fmt=2), "format")
    _refused(call(dtype=7), "dtype")
    _refused(call(tile=24), "tile")
    _refused(call(rows=-1), "row count")
    _refused(call(rows=5), "5 rows of 4")
    _refused(call(ldx=63), "source rows")
    _refused(call(q=P + 8), "16-byte")
    _refused(call(ldq=24), "16-byte")
    _refused(call(sf=P + 4), "16-byte")
    _refused(call(x=P + 1), "misaligned")
    _refused(call(x=None), "null")
    _refused(call(ids=P, div=0), "id_div")
    _refused(call(fmt=0, g=P), "no factor")


def test_dequantize_and_pack_refusals():
    def call(q=P, ldq=32, sf=P, fmt=0, tile=16, rows=4, K=64, g=None, out=P, dtype=0, ldo=64):
        return L.lib().fus_fp4_dequantize(q, ldq, sf, fmt, tile, rows, K, g, 0, out, dtype, ldo, None, None)

    assert call(rows=0) == 0
    _refused(call(ldo=63), "output rows")
    _refused(call(ldq=28), "8-byte")
    _refused(call(g=P), "no factor")
    _refused(call(out=None), "null")
    _refused(L.lib().fus_fp4_pack_scales(P, 0, 2, 32, 33, 0, P, None), "sizes")
    _refused(L.lib().fus_fp4_pack_scales(None, 0, 2, 32, 64, 0, P, None), "null")


def test_gemm_refusals():
    def desc(**kw):
        d = L.Fp4GemmDesc(wq=P, wsf=P, n_experts=2, w_rows=64, K=64, fmt=1, xq=P, ldxq=32, xsf=P,
                          x_rows=32, block_n=16, expert_ids=P, ntp=P, live_ids=P, live_limit=20,
                          scatter=1, epilogue=0, out=P, ldo=64, out_rows=20, out_dtype=0)
        for k, v in kw.items():
            setattr(d, k, v)
        return d

    def call(**kw):
        return L.lib().fus_fp4_grouped_gemm(ctypes.byref(desc(**kw)), None, None)

    assert call(x_rows=0) == 0 and call(out_rows=0) == 0
    for kw, text in (({"K": 48}, "multiple of 32"), ({"w_rows": 40}, "multiple of 16"),
                     ({"block_n": 48}, "block_n"), ({"epilogue": 2}, "epilogue"), ({"fmt": 3}, "format"),
                     ({"out_dtype": 2}, "output is"), ({"wq": None}, "null"), ({"xsf": P + 8}, "aligned"),
                     ({"ldo": 56}, "output rows"), ({"ldo": 68}, "output rows"),
                     ({"live_ids": None}, "live_ids"), ({"expert_ids": None}, "expert_ids"),
                     ({"n_experts": 0}, "n_experts"), ({"fmt": 0, "xg": P}, "no factors"),
                     ({"ldxq": 16}, "aligned"), ({"x_rows": -1}, "row counts")):
        _refused(call(**kw), text)
    d = desc(live_ids=None, scatter=0)
    _refused(L.lib().fus_fp4_expert_gemm(ctypes.byref(d), P, 0, 64, 4, 8, None, None, None), "live_ids")
    _refused(L.lib().fus_fp4_expert_gemm(None, P, 0, 64, 4, 8, None, None, None), "null descriptor")


def test_python_refusals():
    q = torch.zeros(2, 32, 32, dtype=torch.uint8)
    s = torch.zeros(2, 32, 2, dtype=torch.uint8)
    for bad in (dict(fmt="fp8"), dict(scales=s[:, :, :1]), dict(q=q.int()), dict(q=q[0]),
                dict(q=q[:, :24]), dict(q=q[:, :, :20])):
        with pytest.raises((ValueError, TypeError)):
            fp4.ExpertGemmFP4(**{"q": q, "scales": s, "fmt": "mx", **bad})
    x = torch.zeros(4, 64)
    ok = (torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4096, dtype=torch.uint8))
    with pytest.raises(ValueError, match="CUDA"):
        ops.fp4_quantize(x, *ok, "mx")
    with pytest.raises(TypeError):
        ops.fp4_quantize(x.int(), *ok, "mx")
    with pytest.raises(ValueError):
        ops.fp4_quantize(x, ok[0][:, :31], ok[1], "mx")
    with pytest.raises(ValueError):
        ops.fp4_quantize(x, ok[0], ok[1][:8], "mx")
    with pytest.raises(ValueError):
        ops.fp4_quantize(x.T, *ok, "mx")


def test_sizes_past_32_bits_are_refused():
    """Counts are C ints: what would wrap around is refused before anything else is looked at."""
    huge, wide = torch.zeros(1, 64).expand(2 ** 32, 64), torch.zeros(4, 1).expand(4, 2 ** 32)
    q, sf = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4096, dtype=torch.uint8)
    for x in (huge, wide):
        with pytest.raises(ValueError, match="too large"):
            ops.fp4_quantize(x, q, sf, "mx")
        with pytest.raises(ValueError, match="too large"):
            ops.fp4_dequantize(q, sf, x, "mx")
        with pytest.raises(ValueError, match="too large"):
            ops.norm_gate_residual(x, x, x)
        with pytest.raises(ValueError, match="too large"):
            ops.route_topk(x, torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int32))


def test_no_live_rows():
    """An empty batch has ids (all pads) and no source: nothing to do, nothing refused."""
    def call(x, x_rows, div, limit):
        return L.lib().fus_fp4_quantize(x, 0, 64, x_rows, 64, 1, None, 0, P, div, limit, None, 16, 16,
                                        P, 32, P, None, None)

    assert call(None, 0, 8, 0) == 0 and call(P, 4, 1, 0) == 0
    _refused(call(None, 0, 8, 8), "null")
    _refused(call(P, 0, 8, 8), "source rows")
    with pytest.raises(ValueError, match="ntp"):
        ops.fp4_quantize(torch.zeros(4, 64), torch.zeros(4, 32, dtype=torch.uint8),
                         torch.zeros(4096, dtype=torch.uint8), "mx", ntp=torch.zeros(0, dtype=torch.int32))


@pytest.mark.parametrize("dense", [True, False])
def test_workspace_outlives_the_launches(monkeypatch, dense):
    """The packed rows belong to a call until its kernels are on the stream: memory that went back
    to the allocator before could be given to another thread's call on the same stream."""
    made, seen = [], []

    class Torch:
        def __getattr__(self, name):
            return getattr(torch, name)

        @staticmethod
        def empty(*args, **kw):
            t = torch.empty(*args, **kw)
            made.append((weakref.ref(t), t.data_ptr()))
            return t

    def launch(dev, name, desc, *args):
        d = L.Fp4GemmDesc.from_address(desc)
        seen.append([r() is not None and p == d.xq for r, p in made])

    g = fp4.ExpertGemmFP4.__new__(fp4.ExpertGemmFP4)  # host tensors: nothing is launched
    g.E, g.K, g.cols, g.fmt, g.device, g._dev = 1, 64, 32, "nv", torch.device("cpu"), -1
    g._desc = L.Fp4GemmDesc(K=64, ldxq=32)
    monkeypatch.setattr(fp4, "torch", Torch())
    monkeypatch.setattr(ops, "_call_on", launch)
    x, out = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(4, 32, dtype=torch.bfloat16)
    if dense:
        g(x, out)
    else:
        i = lambda n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
        g(x, out, i(16), i(1), i(1), 16)
    assert seen == [[True]]


def test_rows_that_the_last_cta_would_count_past_32_bits():
    top = 0x7FFF0000  # the last allowed count; its launch is not tried here
    for rows in (top + 1, 2 ** 31 - 1):
        _refused(L.lib().fus_fp4_quantize(P, 0, 64, 4, 64, 1, None, 0, P, 1, 4, None, rows, 16, P, 32, P,
                                          None, None), "row count")
        _refused(L.lib().fus_fp4_dequantize(P, 32, P, 1, 16, rows, 64, None, 0, P, 0, 64, None, None), "row count")
        d = L.Fp4GemmDesc(wq=P, wsf=P, n_experts=1, w_rows=64, K=64, fmt=1, xq=P, ldxq=32, xsf=P, x_rows=rows,
                          block_n=16, out=P, ldo=64, out_rows=20)
        _refused(L.lib().fus_fp4_grouped_gemm(ctypes.byref(d), None, None), "row counts")
        _refused(L.lib().fus_fp4_expert_gemm(ctypes.byref(d), P, 0, 64, 4, 0, None, None, None), "row counts")
    # and tiles: rows in blocks times the weight's tiles
    d.x_rows, d.w_rows, d.ldo = 2 ** 27, 2 ** 15, 2 ** 15
    _refused(L.lib().fus_fp4_grouped_gemm(ctypes.byref(d), None, None), "too many tiles")


def test_expert_product_without_pairs_launches_nothing():
    """The product starts while its quantiser runs; without one there is nothing it may overlap."""
    d = L.Fp4GemmDesc(wq=P, wsf=P, n_experts=2, w_rows=64, K=64, fmt=1, xq=P, ldxq=32, xsf=P, x_rows=32,
                      block_n=16, expert_ids=P, ntp=P, live_ids=P, live_limit=0, scatter=1, out=P, ldo=64, out_rows=20)
    for rows, div in ((0, 8), (4, 8), (4, 1)):
        assert L.lib().fus_fp4_expert_gemm(ctypes.byref(d), P, 0, 64, rows, div, P, None, None) == 0
