"""The MoE block with 4-bit experts: each step against 64 bits on the kernel's own inputs of that
step (so that one bf16 rounding before a quantisation does not count twice), and the whole
against the steps."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import fp4_oracle as Q
from fusion_b200 import fp4, ops
from fusion_b200.block import MoEBlockFP4
from gpu_util import finish
from test_gpu_fp4 import _reference

pytestmark = pytest.mark.gpu


def _weights(E, H, I, fmt, shared, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    q = lambda *s: fp4.quantize_weight((0.05 * r(*s)).to(torch.bfloat16), fmt)  # noqa: E731
    return dict(gamma=(1 + 0.1 * r(H)).to(torch.bfloat16), gate_w=0.05 * r(E, H), bias=0.01 * r(E),
                w13=q(E, 2 * I, H), w2=q(E, H, I), fmt=fmt,
                w13s=q(1, 2 * I, H) if shared else None, w2s=q(1, H, I) if shared else None)


def _value(w, fmt):
    g = w[2].double().cpu().numpy()[:, None, None] if w[2] is not None else 1.0
    return Q.values(Q.unpack(w[0].cpu().numpy()), w[1].cpu().numpy(), fmt, g)


def _np(t):
    return t.double().cpu().numpy()


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("T,E,H,I,topk,shared,kw", [
    (1, 128, 512, 128, 8, True, {}),
    (5, 128, 256, 96, 4, False, {"score": "softmax", "renorm": False, "routed_scale": 1.0}),
    (40, 128, 512, 160, 8, True, {"n_group": 8, "topk_group": 4}),
    (300, 128, 256, 128, 6, False, {}),
    (700, 128, 256, 64, 8, True, {"residual_scale": 0.5})])
def test_steps(fmt, T, E, H, I, topk, shared, kw):
    w = _weights(E, H, I, fmt, shared)
    g = torch.Generator(device="cuda").manual_seed(T)
    h, r = (torch.randn(T, H, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
    post, nxt = ((1 + 0.1 * torch.randn(H, device="cuda", generator=g)).to(torch.bfloat16) for _ in range(2))
    blk = MoEBlockFP4(**w, topk=topk, post_gamma=post, next_gamma=nxt, **kw)
    blk.calibrate(h, r)
    o = blk(h, r)
    h1, x2, topw, topi, layout, bn = blk._route(h, r)
    act, y, sh = blk._experts(x2, topi, layout, bn)
    merged = torch.empty_like(h1)
    ops.merge(y, topw, None, sh, merged, round_mid=False)
    finish()
    assert torch.equal(o.topi, topi) and torch.equal(o.h1, h1)
    # layout: every pair once
    ids = layout[0][: int(layout[2].item())].cpu().numpy()
    live = np.flatnonzero(ids < T * topk)
    np.testing.assert_array_equal(np.sort(ids[live]), np.arange(T * topk))
    # w13 + SwiGLU on the block's x2, w2 on its act
    sx = [float(s.item()) if s is not None else 1.0 for s in blk.x_scales]
    ti = topi.cpu().numpy()
    xq = Q.values(*Q.quantize(_np(x2), fmt, sx[0]), fmt, sx[0])
    want, err = _reference(xq, _value(w["w13"], fmt), ti, True)
    got = _np(act)[live]
    ref, e = want[ids[live]], err[ids[live]]
    assert (np.abs(got - ref) <= e + (2.0 ** -8 + 2.0 ** -23) * np.abs(ref) + 1e-30).all()
    a_pair = np.empty((T * topk, I))
    a_pair[ids[live]] = got
    aq = Q.values(*Q.quantize(a_pair, fmt, sx[1]), fmt, sx[1])
    w2 = _value(w["w2"], fmt)
    e2 = ti.reshape(-1)
    ref = np.stack([w2[e] @ v for e, v in zip(e2, aq)])
    mag = np.stack([np.abs(w2[e]) @ np.abs(v) for e, v in zip(e2, aq)])
    bound = (I / 16 + 4) * 2.0 ** -23 * mag + (2.0 ** -8 + 2.0 ** -23) * np.abs(ref) + 1e-30
    assert (np.abs(_np(y).reshape(T * topk, H) - ref) <= bound).all()
    # shared expert (fp32 out)
    if shared:
        one = np.zeros((T, 1), dtype=int)
        a_s = torch.empty(T, I, dtype=torch.bfloat16, device="cuda")
        blk.w13s(x2, a_s)
        finish()
        want, err = _reference(xq, _value(w["w13s"], fmt), one, True)
        assert (np.abs(_np(a_s) - want) <= err + (2.0 ** -8 + 2.0 ** -23) * np.abs(want) + 1e-30).all()
        aq = Q.values(*Q.quantize(_np(a_s), fmt, sx[1]), fmt, sx[1])
        ws = _value(w["w2s"], fmt)[0]
        ref, mag = aq @ ws.T, np.abs(aq) @ np.abs(ws).T
        assert (np.abs(_np(sh) - ref) <= (I / 16 + 8) * 2.0 ** -23 * mag + 1e-30).all()
    # merge, then norm + residual + next norm
    ref = (_np(topw)[..., None] * _np(y)).sum(1) + (_np(sh) if shared else 0.0)
    mag = (np.abs(_np(topw))[..., None] * np.abs(_np(y))).sum(1) + (np.abs(_np(sh)) if shared else 0.0)
    assert (np.abs(_np(merged) - ref) <= 2.0 ** -8 * np.abs(ref) + 2.0 ** -20 * mag).all()
    out, x = torch.empty_like(h1), torch.empty_like(h1)
    ops.norm_gate_residual(merged, h1, out, x, post_w=post, pre_w=nxt, alpha=kw.get("residual_scale", 1.0))
    finish()
    assert torch.equal(out, o.out) and torch.equal(x, o.x)


def test_without_norms_and_masked_router():
    """No norms after the block: the residual goes into the merge. A router that masks all but two
    experts leaves slots empty; they add nothing."""
    E, H, I, topk, T = 128, 256, 64, 4, 9
    w = _weights(E, H, I, "mx", False)
    blk = MoEBlockFP4(**(w | {"bias": None}), topk=topk)
    h, r = (torch.randn(T, H, device="cuda").to(torch.bfloat16) for _ in range(2))
    o = blk(h, r)
    h1, x2, topw, topi, layout, bn = blk._route(h, r)
    _, y, _ = blk._experts(x2, topi, layout, bn)
    finish()
    ref = (_np(topw)[..., None] * _np(y)).sum(1) + _np(h1)
    mag = (np.abs(_np(topw))[..., None] * np.abs(_np(y))).sum(1) + np.abs(_np(h1))
    assert o.x is None and (np.abs(_np(o.out) - ref) <= 2.0 ** -8 * np.abs(ref) + 2.0 ** -20 * mag).all()
    # every expert but 3 and 7 masked
    logits = torch.full((T, E), -float("inf"), device="cuda")
    logits[:, 3], logits[:, 7] = 1.0, 2.0
    ops.route_topk(logits, topw, topi)
    sorted_ids, eids, ntp = (torch.empty(n, dtype=torch.int32, device="cuda") for n in (T * topk + E * 15, (T * topk + E * 15) // 16, 1))
    cap = sorted_ids.numel() // 16 * 16
    ops.moe_align(topi, E, 16, sorted_ids[:cap], eids, ntp)
    # rows that nothing writes must not be what memory held: fill the pool with NaN first
    junk = [torch.full((T * topk, H), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(4)]
    del junk
    _, y, _ = blk._experts(x2, topi, (sorted_ids[:cap], eids, ntp), 16)
    finish()
    assert (topi[:, :2].cpu() == torch.tensor([7, 3])).all() and (topi[:, 2:] == -1).all()
    assert (y[:, 2:] == 0).all() and (y[:, :2].abs().amax(-1) > 0).all()


@pytest.mark.parametrize("T", [1, 33])
def test_graph_on_another_stream(T):
    w = _weights(128, 512, 128, "nv", True)
    blk = MoEBlockFP4(**w, next_gamma=w["gamma"])
    hs = [torch.randn(T, 512, device="cuda").to(torch.bfloat16) for _ in range(4)]
    blk.calibrate(hs[0], hs[1])
    want = [blk(hs[0], hs[1]), blk(hs[2], hs[3])]
    h, r = hs[0].clone(), hs[1].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = blk(h, r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in (0, 1, 0, 1):
            h.copy_(hs[2 * i]), r.copy_(hs[2 * i + 1])
            graph.replay()
    finish()
    assert torch.equal(o.out, want[1].out) and torch.equal(o.x, want[1].x)


def test_empty_batch():
    w = _weights(128, 256, 64, "mx", True)
    blk = MoEBlockFP4(**w, next_gamma=w["gamma"])
    e = torch.empty(0, 256, dtype=torch.bfloat16, device="cuda")
    o = blk(e, e)
    assert o.out.shape == (0, 256) and o.x.shape == (0, 256)


@pytest.mark.parametrize("times", [0.2, 1.0, 8.0])
def test_calibration_covers_the_shared_expert(times):
    """The shared expert's activations have the routed ones' factor: it holds the largest of both, and
    no block that the down projection reads is cut off. Each value is off by half the widest
    step of its block (1 of a scale, which is a sixth of the largest within 2^-4), by 2^-4 of the
    largest where the scale was rounded down, and by the smallest scale's half step (2^-10)."""
    T, E, H, I, topk = 33, 128, 256, 96, 4
    w = _weights(E, H, I, "nv", True)
    g = torch.Generator(device="cuda").manual_seed(1)
    gate_up = times * 0.05 * torch.randn(1, 2 * I, H, device="cuda", generator=g)
    w["w13s"] = fp4.quantize_weight(gate_up.to(torch.bfloat16), "nv")
    blk = MoEBlockFP4(**w, topk=topk)
    h, r = (torch.randn(T, H, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
    blk.calibrate(h, r)
    _, x2, _, topi, layout, bn = blk._route(h, r)
    act, _, shared = blk._experts(x2, topi, layout, bn)
    act_s = torch.empty(T, I, dtype=torch.bfloat16, device="cuda")
    blk.w13s(x2, act_s)
    finish()
    ids = layout[0][: int(layout[2].item())]
    routed = act[: ids.numel()][ids < T * topk]
    a = _np(act_s)
    factor = float(blk.x_scales[1].item())
    assert factor == float(np.float32(max(float(routed.abs().max()), np.abs(a).max())) / np.float32(2688.0))
    block = np.abs(a).reshape(T, I // 16, 16).max(-1)
    off = np.repeat(np.maximum(block * (1 + 2.0 ** -4) / 6, block * 2.0 ** -4) + 6 * factor * 2.0 ** -10, 16, axis=-1)
    w2s = _value(w["w2s"], "nv")[0]
    bound = off @ np.abs(w2s).T + (I / 16 + 8) * 2.0 ** -23 * ((np.abs(a) + off) @ np.abs(w2s).T) + 1e-30
    assert (np.abs(_np(shared) - a @ w2s.T) <= bound).all()
