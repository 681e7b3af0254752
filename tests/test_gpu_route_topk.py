"""Routing from logits on the GPU against its definition in 64 bits: ids exactly, weights within
the rounding of fp32 sums and exponentials."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from fusion_b200 import ops
from gpu_util import finish

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _oracle(l, bias, score, n_group, topk_group, k, renorm, scale):
    T, E = l.shape
    l = np.where(np.isnan(l), -np.inf, np.minimum(l, np.finfo(np.float32).max))
    with np.errstate(all="ignore"):
        if score == "sigmoid":
            s = 1 / (1 + np.exp(-l))
        else:
            e = np.where(l > -np.inf, np.exp(l - l.max(1, keepdims=True)), 0.0)
            s = e / e.sum(1, keepdims=True)
    c = np.where(l > -np.inf, s + (0.0 if bias is None else bias), -np.inf)
    if n_group > 1:
        g = c.reshape(T, n_group, -1)
        two = -np.sort(-g, -1)[..., :2]
        best = np.where(np.isfinite(two).any(-1), np.where(np.isfinite(two), two, 0.0).sum(-1), -np.inf)
        keep = np.argsort(-best, 1, kind="stable")[:, :topk_group]
        mask = np.zeros((T, n_group), bool)
        np.put_along_axis(mask, keep, True, 1)
        c = np.where(mask[..., None], g, -np.inf).reshape(T, E)
    # a plain choice ranks the logits: the score is monotone in them, and exact
    rank = l if bias is None and n_group == 1 else c
    ids = np.argsort(-rank, 1, kind="stable")[:, :k]
    ok = np.take_along_axis(rank, ids, 1) > -np.inf
    w = np.where(ok, np.take_along_axis(np.nan_to_num(s), ids, 1), 0.0)
    if renorm:
        w = w / np.maximum(w.sum(1, keepdims=True), 1e-20)
    return np.where(ok, ids, -1), w * scale


def _run(logits, k, bias=None, score="sigmoid", n_group=1, topk_group=1, renorm=True, scale=1.0):
    T = logits.shape[0]
    w = torch.full((T, k), 9.0, device="cuda")
    i = torch.full((T, k), 9, dtype=torch.int32, device="cuda")
    ops.route_topk(logits, w, i, score=score, bias=bias, n_group=n_group, topk_group=topk_group,
                   renorm=renorm, scale=scale)
    finish()
    ids, want = _oracle(logits.double().cpu().numpy(), None if bias is None else bias.double().cpu().numpy(),
                        score, n_group, topk_group, k, renorm, scale)
    np.testing.assert_array_equal(i.cpu().numpy(), ids)
    # (E / 32 + 5) roundings of the sum, 25 of an exponential of -20, ten more: below 2^-17
    got = w.double().cpu().numpy()
    assert (np.abs(got - want) <= 2.0 ** -17 * np.abs(want) + 1e-30).all()


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("T,E,k,n_group,topk_group", [
    (1, 256, 8, 1, 1), (1, 1, 1, 1, 1), (7, 8, 8, 1, 1), (33, 33, 5, 1, 1), (130, 162, 6, 1, 1),
    (65, 256, 8, 8, 4), (19, 104, 3, 8, 2), (40, 512, 8, 4, 1), (9, 1024, 32, 1, 1),
    (21, 60, 4, 5, 2), (17, 64, 8, 32, 8), (300, 48, 24, 3, 3), (5, 1000, 10, 1, 1)])
def test_matches_definition(score, dtype, with_bias, T, E, k, n_group, topk_group):
    gen = torch.Generator(device="cuda").manual_seed(T * E + k)
    logits = torch.randn(T, E, device="cuda", generator=gen).to(DTYPES[dtype])
    bias = 0.1 * torch.randn(E, device="cuda", generator=gen) if with_bias else None
    _run(logits, k, bias, score, n_group, topk_group, renorm=bool(E % 3), scale=2.5)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_long_batch(score):
    """Enough rows that some decisions hang on the last bits of fp32 scores."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    logits = 0.02 * torch.randn(20000, 256, device="cuda", generator=gen)
    bias = 1e-4 * torch.randn(256, device="cuda", generator=gen)
    _run(logits, 8, bias, score)
    _run(logits, 8, bias, score, n_group=8, topk_group=4)
    _run(logits, 8, None, score, n_group=8, topk_group=4)


def test_ties_go_to_the_lower_id():
    logits = torch.zeros(4, 200, device="cuda")
    logits[1] = torch.arange(200, device="cuda") // 40
    logits[2, ::7] = 1.0
    logits[3] = 3.0
    for bias in (None, torch.zeros(200, device="cuda"), torch.full((200,), 0.5, device="cuda")):
        for score in ("sigmoid", "softmax"):
            _run(logits, 8, bias, score)
            _run(logits, 8, bias, score, n_group=4, topk_group=2)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("bias", [False, True])
def test_masked_experts_and_empty_rows(score, bias):
    """-inf and NaN mask; rows left with fewer than k experts, with one, with none; the lowest
    finite value is a logit like any other; +inf is the largest."""
    logits = torch.randn(9, 96, device="cuda")
    inf = float("inf")
    logits[0] = -inf
    logits[1] = float("nan")
    logits[2, 1:] = -inf
    logits[3, 5:] = float("nan")
    logits[4, ::2] = -inf
    logits[5] = torch.finfo(torch.float32).min
    logits[6, 3] = inf
    logits[6, 50] = inf
    logits[7, 4:90] = torch.finfo(torch.float32).min
    b = 0.3 * torch.randn(96, device="cuda") if bias else None
    for groups in (1, 4):
        _run(logits, 6, b, score, n_group=groups, topk_group=max(1, groups // 2))


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_scores_that_saturate(score):
    """Logits whose scores are 1 (or 0) in any precision still rank by themselves, also in rows with
    more ties than candidates."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    logits = 40 + 20 * torch.randn(40, 256, device="cuda", generator=gen).round()
    logits[::2] = logits[::2].clamp(0, 60)
    logits[1::4] -= 2000
    logits[3] = 40 + torch.arange(256, device="cuda") % 7
    _run(logits, 8, None, score)
    _run(logits, 20, None, score, renorm=False)


def test_large_bias_and_logits():
    gen = torch.Generator(device="cuda").manual_seed(9)
    logits = 60 * torch.randn(50, 128, device="cuda", generator=gen)
    bias = 100 * torch.randn(128, device="cuda", generator=gen).round()
    _run(logits, 8, bias)
    _run(logits.clamp(-8, 8), 8, -bias, n_group=8, topk_group=3)


def test_strided_logits_and_rows_behind():
    buf = torch.randn(10, 300, device="cuda")
    for off in (0, 1, 4):
        _run(buf[:, off:off + 250], 8, torch.randn(250, device="cuda"))
    w = torch.full((12, 8), 7.0, device="cuda")
    i = torch.full((12, 8), 7, dtype=torch.int32, device="cuda")
    ops.route_topk(buf, w[:10], i[:10])
    finish()
    assert (w[10:] == 7).all() and (i[10:] == 7).all()


def test_stream_graph_and_empty_batch():
    logits = torch.randn(64, 256, device="cuda")
    w, i = torch.empty(64, 8, device="cuda"), torch.empty(64, 8, dtype=torch.int32, device="cuda")
    ops.route_topk(logits, w, i)
    w2, i2 = torch.zeros_like(w), torch.zeros_like(i)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.route_topk(logits, w2, i2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        g.replay()
    finish()
    assert torch.equal(w, w2) and torch.equal(i, i2)
    ops.route_topk(logits[:0], w[:0], i[:0])
    finish()


def test_feeds_the_dispatch_layout():
    """Holes of masked rows are not placed."""
    logits = torch.randn(12, 16, device="cuda")
    logits[3] = -float("inf")
    w, i = torch.empty(12, 4, device="cuda"), torch.empty(12, 4, dtype=torch.int32, device="cuda")
    ops.route_topk(logits, w, i, score="softmax")
    sorted_ids = torch.empty(48 + 16 * 16, dtype=torch.int32, device="cuda")
    eids = torch.empty(19, dtype=torch.int32, device="cuda")
    ntp = torch.empty(1, dtype=torch.int32, device="cuda")
    ops.moe_align(i, 16, 16, sorted_ids, eids, ntp)
    finish()
    placed = sorted_ids[: int(ntp.item())].cpu().numpy()
    assert sorted(placed[placed < 48]) == [p for p in range(48) if p // 4 != 3]


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("E,n_group,topk_group,k", [(64, 8, 4, 4), (256, 8, 4, 8), (160, 5, 2, 6), (96, 32, 7, 6),
                                                    (128, 16, 16, 8), (1024, 2, 1, 9)])
def test_close_groups(score, with_bias, E, n_group, topk_group, k):
    """Groups whose two largest logits differ by a few units in the last place or not at all, groups
    with one expert or none: decided as 64-bit arithmetic decides them."""
    rng = np.random.default_rng(E + n_group)
    T, size = 600, E // n_group
    l = rng.normal(-2.0, 0.5, (T, n_group, size)).astype(np.float32)
    steps = rng.integers(-2, 3, (T, n_group, 2)).astype(np.float32)
    for t in range(T):
        for g in range(n_group):
            at = rng.choice(size, 2, replace=False)
            l[t, g, at[0]] = np.float32(1.25) * (1 + steps[t, g, 0] * 2.0 ** -22)
            l[t, g, at[1]] = np.float32(0.75) * (1 + steps[t, g, 1] * 2.0 ** -22)
    one = rng.random((T, n_group)) < 0.1
    l[np.repeat(one[..., None], size, 2) & (l < 1.0)] = -np.inf  # one expert is left
    l[rng.random((T, n_group)) < 0.1] = -np.inf
    bias = torch.full((E,), 0.125, device="cuda") if with_bias else None
    _run(torch.from_numpy(l.reshape(T, E)).cuda(), k, bias, score, n_group, topk_group)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("size", [8, 32])
@pytest.mark.parametrize("topk_group", [1, 2, 4])
@pytest.mark.parametrize("large,step", [(100.0, 1e-4), (1000.0, 1e-4), (1000.0, 1e-3), (10000.0, 1e-2)])
def test_groups_whose_choices_cancel(score, size, topk_group, large, step):
    """Biases of either sign: a group's two largest choices are large, their sum is not. fp32 cannot
    tell such sums apart where their magnitudes' last places are, whatever the sum's are."""
    gen = torch.Generator(device="cuda").manual_seed(size)
    T, G = 500, 8
    # scores some `step` apart: a softmax's are smaller by the number of experts
    step *= 0.24 * G * size if score == "softmax" else 1.0
    logits = 0.3 + step * torch.randn(T, G * size, device="cuda", generator=gen)
    bias = torch.full((G, size), -large, device="cuda")
    bias[:, 2] = large
    _run(logits, topk_group, bias.reshape(-1), score, n_group=G, topk_group=topk_group)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("groups", [1, 4])
@pytest.mark.parametrize("k", [1, 3])
@pytest.mark.parametrize("first,out", [((), (0, 9, 63)), ((5,), ()), ((40, 7), (3,)), ((50, 40, 7, 8), ()),
                                       ((1, 2, 17, 18, 19, 30, 31), (0, 3))])
def test_infinite_bias(score, groups, k, first, out):
    """A bias of +infinity puts an expert first (several: the lower id), of -infinity leaves it out."""
    gen = torch.Generator(device="cuda").manual_seed(len(first))
    T, E = 70, 64
    logits = torch.randn(T, E, device="cuda", generator=gen)
    bias = 0.1 * torch.randn(E, device="cuda", generator=gen)
    bias[list(first)], bias[list(out)] = float("inf"), -float("inf")
    w = torch.full((T, k), 9.0, device="cuda")
    i = torch.full((T, k), 9, dtype=torch.int32, device="cuda")
    topk_group = max(1, groups // 2)
    ops.route_topk(logits, w, i, score=score, bias=bias, n_group=groups, topk_group=topk_group)
    finish()
    e = np.exp(logits.double().cpu().numpy())
    s = e / (1 + e) if score == "sigmoid" else e / e.sum(1, keepdims=True)
    c = (s + bias.double().cpu().numpy()).reshape(T, groups, -1)
    best = -np.sort(-c, -1)[..., :2].sum(-1)
    drop = np.argsort(-best, 1, kind="stable")[:, topk_group:]
    np.put_along_axis(c, drop[..., None], -np.inf, 1)
    ids = np.argsort(-c.reshape(T, E), 1, kind="stable")[:, :k]
    want = np.take_along_axis(s, ids, 1)
    want /= want.sum(1, keepdims=True)
    np.testing.assert_array_equal(i.cpu().numpy(), ids)
    assert (np.abs(w.double().cpu().numpy() - want) <= 2.0 ** -17 * want).all()
