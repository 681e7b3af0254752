"""What the routing and the block norms refuse, on the host."""

from __future__ import annotations

import contextlib
import weakref
from types import SimpleNamespace

import pytest
import torch

from fusion_b200 import _lib as L
from fusion_b200 import ops

P = 0x10000  # an aligned address that host checks never read


def _refused(rc, text):
    assert rc in (-1, -3) and text in L.last_error(), L.last_error()


def test_route_topk():
    def call(logits=P, dtype=1, ld=64, bias=None, score=0, n_group=1, topk_group=1, topw=P, topi=P,
             T=4, E=64, k=8):
        return L.lib().fus_route_topk(logits, dtype, ld, bias, score, n_group, topk_group, topw, topi,
                                      T, E, k, 1.0, 1, None, None)

    assert call(T=0) == 0
    _refused(call(k=33), "topk")
    _refused(call(k=0), "topk")
    _refused(call(E=4), "topk")
    _refused(call(T=-1), "T=-1")
    _refused(call(dtype=3), "dtype")
    _refused(call(score=2), "score")
    _refused(call(n_group=5), "n_group")
    _refused(call(n_group=64), "n_group")
    _refused(call(n_group=4, topk_group=5), "topk_group")
    _refused(call(n_group=16, topk_group=1), "fewer than topk")
    _refused(call(E=1056, ld=1056), "too many experts")
    _refused(call(ld=63), "logit rows")
    _refused(call(logits=P + 2), "logit rows")
    _refused(call(topi=None), "null")


def test_norm_gate_residual():
    def call(y=P, ldy=64, res=P, post_w=None, gate=None, ldg=0, kind=0, act=0, h=P, pre_w=None, x=None,
             ldx=64, T=4, N=64, dtype=0):
        return L.lib().fus_norm_gate_residual(y, ldy, res, 64, post_w, gate, ldg, kind, act, 1.0, h, 64,
                                              pre_w, x, ldx, T, N, dtype, 1e-5, None, None)

    assert call(T=0) == 0
    _refused(call(N=0), "sizes")
    _refused(call(dtype=5), "dtype")
    _refused(call(kind=4, gate=P), "gate")
    _refused(call(act=3), "gate")
    _refused(call(kind=2), "null")
    _refused(call(x=P), "go together")
    _refused(call(pre_w=P), "go together")
    _refused(call(ldy=63), "overlap")
    _refused(call(kind=3, gate=P, ldg=8), "overlap")
    _refused(call(y=P + 1), "misaligned")
    _refused(call(y=None), "null")


def test_clear_holes():
    def call(ids=P, n=4, y=P, ldy=64, H=64):
        return L.lib().fus_clear_holes(ids, n, y, ldy, H, None)

    assert call(n=0) == 0
    _refused(call(n=-1), "sizes")
    _refused(call(H=60), "sizes")
    _refused(call(y=P + 8), "aligned")
    _refused(call(ldy=56), "aligned")
    _refused(call(ids=None), "aligned")
    with pytest.raises(TypeError):
        ops.clear_holes(torch.zeros(4, 64), torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.clear_holes(torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32))


def test_python_refusals():
    x = torch.zeros(4, 64)
    w, i = torch.zeros(4, 8), torch.zeros(4, 8, dtype=torch.int32)
    for args, kw in (((x, w, i), {}), ((x.int(), w, i), {}), ((x, w[:, :4], i), {}), ((x, w, i.long()), {}),
                     ((x, w, i), {"bias": torch.zeros(63)}), ((x.T, w, i), {})):
        with pytest.raises((ValueError, TypeError)):
            ops.route_topk(*args, **kw)
    for args, kw in (((x, x, x), {}), ((x, x.half(), x), {}), ((x, x[:2], x), {}),
                     ((x, x, x), {"post_w": torch.zeros(32)}), ((x, x, x), {"gate": torch.zeros(4, 2)}),
                     ((x, x, x), {"gate": torch.zeros(4, 1).half()}), ((x.T, x.T, x.T), {})):
        with pytest.raises((ValueError, TypeError)):
            ops.norm_gate_residual(*args, **kw)


def test_rows_that_the_last_cta_would_count_past_32_bits():
    for n in (0x7FFF0001, 2 ** 31 - 1):
        _refused(L.lib().fus_route_topk(P, 1, 64, None, 0, 1, 1, P, P, n, 64, 8, 1.0, 1, None, None), f"T={n}")
        _refused(L.lib().fus_clear_holes(P, n, P, 64, 64, None), "sizes")


def test_one_status_word_for_two_first_calls(monkeypatch):
    """Two threads that find no status word make one each; both go on with the first, whose address
    kernels may have by then."""
    first, late = torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)

    def zeros(*args, **kw):
        ops._status[7] = first  # the other thread's, meanwhile
        return late

    monkeypatch.setattr(torch.cuda, "Stream", lambda dev: SimpleNamespace(synchronize=lambda: None))
    monkeypatch.setattr(torch.cuda, "stream", contextlib.nullcontext)
    monkeypatch.setattr(ops.C, "CDLL", lambda name: SimpleNamespace(cuThreadExchangeStreamCaptureMode=lambda m: 0))
    monkeypatch.setattr(ops, "_status", {})
    monkeypatch.setattr(torch, "zeros", zeros)
    assert ops.status_tensor(7) is first and ops._status[7] is first


@pytest.mark.parametrize("entry", [ops.router_split_weight, ops.router_transpose_weight])
def test_copied_weights_outlive_the_launch(monkeypatch, entry):
    """A router weight that is copied to be contiguous: the copy is there when the kernel is launched."""
    passed, alive = [], []
    address = ops._p
    monkeypatch.setattr(ops, "_p", lambda t: passed.append(weakref.ref(t)) or address(t))
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(L, "call", lambda *args: alive.extend(r() is not None for r in passed))
    entry(torch.zeros(8, 16).T)
    assert alive == [True, True]
