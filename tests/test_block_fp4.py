"""The 4-bit MoE block's host side: the device its calls run on and what it refuses."""

from __future__ import annotations

import contextlib
from types import SimpleNamespace

import pytest
import torch

from fusion_b200 import fp4, ops
from fusion_b200.block import MoEBlockFP4

E, H, I = 4, 64, 32


@pytest.fixture
def current(monkeypatch):
    """The devices made current, innermost last."""
    stack = []

    @contextlib.contextmanager
    def device(d):
        stack.append(d)
        yield
        stack.pop()

    monkeypatch.setattr(torch.cuda, "device", device)
    return stack


def _block(monkeypatch, **kw):
    """A block on the host: projections that only know their sizes, nothing is launched."""
    def projection(q, scales, fmt, gscale=None, x_gscale=None, gate_up=False):
        return SimpleNamespace(E=q.shape[0], N=q.shape[1], K=2 * q.shape[2], gate_up=gate_up,
                               cols=q.shape[1] // 2 if gate_up else q.shape[1])

    monkeypatch.setattr(fp4, "ExpertGemmFP4", projection)
    stack = lambda e, n, k: (torch.zeros(e, n, k // 2, dtype=torch.uint8), None, None)  # noqa: E731
    args = dict(gamma=torch.ones(H, dtype=torch.bfloat16), gate_w=torch.zeros(E, H), bias=None,
                w13=stack(E, 2 * I, H), w2=stack(E, H, I), fmt="nv")
    return MoEBlockFP4(**(args | {k: stack(*v) if k in ("w13", "w2", "w13s", "w2s") else v for k, v in kw.items()}))


def test_every_launch_is_under_the_blocks_device(monkeypatch, current):
    class Reached(Exception):
        pass

    def launch(*args, **kw):
        raise Reached(list(current))

    monkeypatch.setattr(ops, "router_split_weight", launch)
    with pytest.raises(Reached) as got:
        _block(monkeypatch)
    assert got.value.args[0] == [torch.device("cpu")]
    del current[:]
    monkeypatch.setattr(ops, "router_split_weight", lambda w: torch.zeros(E, 3 * H, dtype=torch.bfloat16))
    blk = _block(monkeypatch)
    blk._route = launch
    h = torch.zeros(2, H, dtype=torch.bfloat16)
    for call in (blk.forward, blk.calibrate):
        del current[:]
        with pytest.raises(Reached) as got:
            call(h, h)
        assert got.value.args[0] == [blk.device]


@pytest.mark.parametrize("call", ["forward", "calibrate"])
def test_inputs_that_do_not_fit_are_refused(monkeypatch, current, call):
    """Nothing past the end of h or r is read: both are [T, H] bf16 on the block's device."""
    monkeypatch.setattr(ops, "router_split_weight", lambda w: torch.zeros(E, 3 * H, dtype=torch.bfloat16))
    blk = _block(monkeypatch)
    blk._route = lambda *a: pytest.fail("launched")
    h = torch.zeros(4, H, dtype=torch.bfloat16)
    for a, b in ((h, h[:3]), (h[:3], h), (h[:, :32], h[:, :32]), (h[0], h[0]), (h, h[:, :32]), (h[None], h[None]),
                 (h.view(2, 2 * H)[:, ::2], h[:2]), (h, h.to("meta")), (h.to("meta"), h.to("meta"))):
        with pytest.raises(ValueError):
            getattr(blk, call)(a, b)
    for a, b in ((h.float(), h), (h, h.half())):
        with pytest.raises(TypeError):
            getattr(blk, call)(a, b)


def test_weights_that_do_not_fit_are_refused(monkeypatch, current):
    """Nothing past the end of a norm's weights or the bias is read, no projection of another size is
    taken."""
    monkeypatch.setattr(ops, "router_split_weight", lambda w: torch.zeros(*w.shape[:1], 3 * w.shape[1]))
    one = torch.ones(H, dtype=torch.bfloat16)
    good = _block(monkeypatch, w13s=(1, 2 * I, H), w2s=(1, H, I), post_gamma=one, next_gamma=one,
                  bias=torch.zeros(E), x_scales=(torch.ones(1), torch.ones(1)))
    assert (good.E, good.H, good.I) == (E, H, I)
    half = _block(monkeypatch, x_scales=(torch.full((1,), 3.0), None))  # no factor: 1
    assert [float(s) for s in half.x_scales] == [3.0, 1.0]
    for bad in ({"gamma": one[:32]}, {"post_gamma": one[:32]}, {"next_gamma": torch.ones(2 * H, dtype=torch.bfloat16)[::2]},
                {"bias": torch.zeros(E - 1)}, {"bias": torch.zeros(E, device="meta")},
                {"w13": (E, 2 * I, 2 * H)}, {"w13": (E + 1, 2 * I, H)}, {"w2": (E, H, 2 * I)}, {"w2": (E, 2 * H, I)},
                {"w13s": (1, 2 * I, H)}, {"w13s": (2, 2 * I, H), "w2s": (1, H, I)},
                {"w13s": (1, 4 * I, H), "w2s": (1, H, 2 * I)}, {"w13s": (1, 2 * I, H), "w2s": (1, 2 * H, I)},
                {"x_scales": (torch.ones(1),)}):
        with pytest.raises(ValueError):
            _block(monkeypatch, **bad)
    for bad in ({"gamma": one.float()}, {"post_gamma": one.half()}, {"bias": torch.zeros(E).half()},
                {"gate_w": torch.zeros(E, H).half()}, {"gate_w": torch.zeros(H)}):
        with pytest.raises(TypeError):
            _block(monkeypatch, **bad)
