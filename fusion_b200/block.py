"""The GLM-5.2 MoE block on one GPU: weights, workspace and the forward call.

``MoEBlock.forward`` is one call into ``fus_moe_block_forward`` (8 kernel launches, no
host synchronisation, see ``csrc/block.cu``). ``MoEBlock.capture`` records that call
in a CUDA graph for a fixed T, which removes the per-launch host cost at decode sizes.

Reference: the block as glm52/bench/bench_layer.py:365-374 composes it, chained like
build_chain (bench_layer.py:395-481) without o_proj.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from . import _lib as L
from . import fp4, ops


@dataclass
class BlockOutputs:
    out: torch.Tensor    # [T, H] bf16  = h1 + routed + shared
    h1: torch.Tensor     # [T, H] bf16  new residual
    topw: torch.Tensor   # [T, k] fp32
    topi: torch.Tensor   # [T, k] int32


class MoEBlock:
    """Holds device weights in the reference's layouts:
    gamma [H] bf16, gate_w [E,H] fp32 (or bf16), bias [E] fp32 | None,
    w13 [E,2I,H] bf16, w2 [E,H,I] bf16, shared w13s [2I,H] / w2s [H,I] bf16 | None.
    n_group / topk_group > 1 select noaux_tc grouped routing (DeepSeek-V3-style)."""

    def __init__(self, gamma, gate_w, bias, w13, w2, w13s=None, w2s=None, *, topk: int = 8,
                 eps: float = 1e-5, routed_scale: float = 2.5, renorm: bool = True,
                 n_group: int = 1, topk_group: int = 1):
        self.E, twoI, self.H = w13.shape
        self.I = twoI // 2
        self.topk = topk
        self.device = w13.device
        if gate_w.dtype == torch.float32:
            self.wa, self.nplanes = ops.router_split_weight(gate_w), 3
        else:
            self.wa, self.nplanes = gate_w.contiguous(), 1
        self._keep = [gamma, bias, w13, w2, w13s, w2s, self.wa]
        d = L.BlockDesc()
        d.H, d.I, d.E, d.topk = self.H, self.I, self.E, topk
        d.eps, d.routed_scale, d.renorm = eps, routed_scale, int(renorm)
        d.gamma = gamma.data_ptr()
        d.wa = self.wa.data_ptr()
        d.nplanes = self.nplanes
        d.bias = bias.data_ptr() if bias is not None else None
        d.w13, d.w2 = w13.data_ptr(), w2.data_ptr()
        d.w13s = w13s.data_ptr() if w13s is not None else None
        d.w2s = w2s.data_ptr() if w2s is not None else None
        d.n_group, d.topk_group = n_group, topk_group  # noaux_tc grouping (1: GLM-5.2)
        d.flags = 0
        self.desc = d
        self._ws: torch.Tensor | None = None
        self._graphs: dict[int, tuple] = {}

    # ------------------------------------------------------------------------------
    def block_n(self, T: int) -> int:
        return int(L.lib().fus_moe_block_pick_block_n(T, self.E, self.topk))

    def workspace_bytes(self, T: int, block_n: int = 0) -> int:
        return int(L.lib().fus_moe_block_workspace(ctypes.byref(self.desc), T, block_n))

    def _workspace(self, nbytes: int) -> torch.Tensor:
        # zero once: the block keeps its counters zero between calls
        if self._ws is None or self._ws.numel() < nbytes:
            self._ws = torch.zeros(nbytes, dtype=torch.uint8, device=self.device)
        return self._ws

    def alloc_outputs(self, T: int) -> BlockOutputs:
        dev = self.device
        return BlockOutputs(
            out=torch.empty(T, self.H, dtype=torch.bfloat16, device=dev),
            h1=torch.empty(T, self.H, dtype=torch.bfloat16, device=dev),
            topw=torch.empty(T, self.topk, dtype=torch.float32, device=dev),
            topi=torch.empty(T, self.topk, dtype=torch.int32, device=dev),
        )

    def forward(self, h: torch.Tensor, r: torch.Tensor, outs: BlockOutputs | None = None,
                block_n: int = 0, workspace: torch.Tensor | None = None) -> BlockOutputs:
        T = h.shape[0]
        assert h.is_contiguous() and r.is_contiguous() and h.shape == (T, self.H)
        if outs is None:
            outs = self.alloc_outputs(T)
        if T == 0:  # an empty batch: nothing to compute
            return outs
        nbytes = self.workspace_bytes(T, block_n)
        ws = workspace if workspace is not None else self._workspace(nbytes)
        L.call("fus_moe_block_forward", ctypes.byref(self.desc), h.data_ptr(), r.data_ptr(), T,
               block_n, outs.out.data_ptr(), outs.h1.data_ptr(), outs.topw.data_ptr(),
               outs.topi.data_ptr(), ws.data_ptr(), ws.numel(),
               torch.cuda.current_stream().cuda_stream, ops.status_tensor().data_ptr())
        return outs

    __call__ = forward

    # ------------------------------------------------------------------------------
    def capture(self, T: int, block_n: int = 0):
        """Record forward() for T tokens in a CUDA graph with static buffers.
        Returns (graph, h_in, r_in, outs): copy inputs into h_in / r_in, replay."""
        if T in self._graphs:
            return self._graphs[T]
        h = torch.zeros(T, self.H, dtype=torch.bfloat16, device=self.device)
        r = torch.zeros_like(h)
        outs = self.alloc_outputs(T)
        ws = torch.zeros(self.workspace_bytes(T, block_n), dtype=torch.uint8, device=self.device)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            self.forward(h, r, outs, block_n, ws)  # warm-up (sets kernel attributes)
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            self.forward(h, r, outs, block_n, ws)
        self._graphs[T] = (g, h, r, outs, ws)
        return self._graphs[T]


@dataclass
class BlockFP4Outputs:
    out: torch.Tensor          # [T, H] bf16  new residual stream
    x: torch.Tensor | None     # [T, H] bf16  input of the next block (with next_gamma)
    h1: torch.Tensor           # [T, H] bf16  h + r
    topw: torch.Tensor         # [T, k] fp32
    topi: torch.Tensor         # [T, k] int32


class MoEBlockFP4:
    """The MoE block with 4-bit expert weights, a router of either score, and optionally the norms
    that some models have around a block:

        h1, x2 = h + r, rmsnorm(h1) * gamma
        topw, topi = route(x2 gate_w^T)                     (ops.route_topk)
        y = sum_k topw_k w2[e_k] (SwiGLU(w13[e_k] x2)) + shared    (quantised rows, fp4.ExpertGemmFP4)
        out = h1 + residual_scale * (rmsnorm(y) * post_gamma | y);  x = rmsnorm(out) * next_gamma

    gamma, post_gamma, next_gamma [H] bf16; gate_w [E, H] fp32 (or bf16); bias [E] fp32 | None; w13 and
    w2, and w13s / w2s of a shared expert (stacks of one), as ``fp4.quantize_weight`` or a
    checkpoint gives them: (codes, scale bytes, factors | None). x_scales: fp32 factors [1] of the
    rows of x2 and of the activations ("nv"; ``calibrate`` sets them from a batch). Expert weights
    take 0.53 ("mx") or 0.56 ("nv") bytes an element instead of 2. No reference counterpart
    beyond the block's own composition (glm52/bench/bench_layer.py:365-374)."""

    def __init__(self, gamma, gate_w, bias, w13, w2, fmt: str, w13s=None, w2s=None, *, topk: int = 8,
                 eps: float = 1e-5, routed_scale: float = 2.5, renorm: bool = True,
                 score: str = "sigmoid", n_group: int = 1, topk_group: int = 1, post_gamma=None,
                 next_gamma=None, residual_scale: float = 1.0, x_scales=None):
        if (w13s is None) != (w2s is None):
            raise ValueError("a shared expert has both projections")
        if gate_w.dim() != 2 or gate_w.dtype not in (torch.float32, torch.bfloat16):
            raise TypeError("gate_w: [E, H] fp32 or bf16 required")
        self.E, self.H = gate_w.shape
        for w, what in ((gamma, "gamma"), (post_gamma, "post_gamma"), (next_gamma, "next_gamma")):
            ops._need(w, torch.bfloat16, what, (self.H,))
        ops._need(bias, torch.float32, "bias", (self.E,))
        self.gamma, self.bias = gamma, bias
        self.device = gamma.device
        for w in (gate_w, bias, post_gamma, next_gamma):
            if w is not None and w.device != self.device:
                raise ValueError(f"tensors on {self.device} and {w.device}")
        if gate_w.dtype == torch.float32:
            with torch.cuda.device(self.device):
                self.wa, self.nplanes = ops.router_split_weight(gate_w), 3
        else:
            self.wa, self.nplanes = gate_w.contiguous(), 1
        self.topk, self.eps, self.routed_scale, self.renorm = topk, eps, routed_scale, renorm
        self.score, self.n_group, self.topk_group = score, n_group, topk_group
        self.post_gamma, self.next_gamma, self.residual_scale = post_gamma, next_gamma, residual_scale
        self.fmt = fmt
        if fmt == "nv":
            x_scales = (None, None) if x_scales is None else x_scales
            if len(x_scales) != 2:
                raise ValueError("x_scales: one factor for the rows of x2, one for the activations")
            x_scales = tuple(torch.ones(1, device=self.device) if s is None else s for s in x_scales)
        self.x_scales = x_scales if fmt == "nv" else (None, None)
        mk = lambda w, i, gate_up: fp4.ExpertGemmFP4(  # noqa: E731
            w[0], w[1], fmt, gscale=w[2], x_gscale=self.x_scales[i], gate_up=gate_up)
        self.w13, self.w2 = mk(w13, 0, True), mk(w2, 1, False)
        self.w13s = mk(w13s, 0, True) if w13s is not None else None
        self.w2s = mk(w2s, 1, False) if w2s is not None else None
        self.I = self.w13.cols
        size = lambda w: (w.E, w.K, w.cols)  # noqa: E731
        if size(self.w13) != (self.E, self.H, self.I) or size(self.w2) != (self.E, self.I, self.H):
            raise ValueError("router, w13 and w2 do not fit together")
        if w13s is not None and (size(self.w13s) != (1, self.H, self.I) or size(self.w2s) != (1, self.I, self.H)):
            raise ValueError("the shared expert's projections do not fit the block's")

    def _empty(self, *shape, dtype=torch.bfloat16):
        return torch.empty(*shape, dtype=dtype, device=self.device)

    def _check(self, h, r) -> None:
        for t, what in ((h, "h"), (r, "r")):
            if t.dtype != torch.bfloat16:
                raise TypeError(f"{what}: bf16 required, not {t.dtype}")
            if t.dim() != 2 or t.shape != (h.shape[0], self.H):
                raise ValueError(f"{what} of shape {tuple(t.shape)}: [T, {self.H}] required, h and r alike")
            ops._rows2d(t, what)
            if t.device != self.device:
                raise ValueError(f"{what} is on {t.device}, the block on {self.device}")

    def _route(self, h, r):
        """Norm, router and dispatch layout: h1, x2, topw, topi, the layout and its block_n."""
        T = h.shape[0]
        h1, x2 = self._empty(T, self.H), self._empty(T, self.H)
        ops.add_rmsnorm(h, r, self.gamma, h1, x2, eps=self.eps)
        nsplit = ops.router_nsplit(T, self.H, self.E, self.nplanes)
        partial = self._empty(nsplit, T, self.E, dtype=torch.float32)
        ops.router_logits(x2, self.wa, self.nplanes, partial, nsplit)
        logits = partial[0]
        if nsplit > 1:
            logits = self._empty(T, self.E, dtype=torch.float32)
            ops.scale_sum_planes(partial, nsplit, None, logits)
        topw = self._empty(T, self.topk, dtype=torch.float32)
        topi = self._empty(T, self.topk, dtype=torch.int32)
        ops.route_topk(logits, topw, topi, score=self.score, bias=self.bias, n_group=self.n_group,
                       topk_group=self.topk_group, renorm=self.renorm, scale=self.routed_scale)
        # The bf16 block's tile. For 4-bit weights too it is the fastest or within 3 % of it (256
        # experts, top-8, w13 + w2, NV us at tiles 16 / 32 / 64 / 128 / 256: T 256 821 832 869 1005
        # 1141, 512 888 863 888 1001 1134, 1024 1242 1039 929 1113 1177, 2048 2183 1435 1193 1219
        # 1303, 4096 - 2308 1704 1765 1415), but for MX at 12 rows an expert (T 384: 842 at 16, 790
        # at 32).
        bn = int(L.lib().fus_moe_block_pick_block_n(T, self.E, self.topk))
        R = T * self.topk
        cap = -(-(R + min(R, self.E) * (bn - 1)) // bn) * bn
        layout = (self._empty(cap, dtype=torch.int32), self._empty(cap // bn, dtype=torch.int32),
                  self._empty(1, dtype=torch.int32))
        # large batches: an expert's rows spread evenly over its blocks
        ops.moe_align(topi, self.E, bn, *layout, flags=ops.ALIGN_BALANCED if T > 16 else 0)
        return h1, x2, topw, topi, layout, bn

    def _experts(self, x2, topi, layout, bn):
        """Rows [T, k, H] of the routed experts and the shared expert's [T, H] (fp32) or None."""
        T = x2.shape[0]
        act = self._empty(layout[0].numel(), self.I)
        self.w13(x2, act, *layout, bn, topk=self.topk, scatter=False)
        y = self._empty(T * self.topk, self.H)
        ops.clear_holes(y, topi)  # a slot without an expert (weight 0) is written by no one else
        self.w2(act, y, *layout, bn, gather=False, pairs=T * self.topk)
        shared = None
        if self.w13s is not None:
            act_s, shared = self._empty(T, self.I), self._empty(T, self.H, dtype=torch.float32)
            self.w13s(x2, act_s)
            self.w2s(act_s, shared)
        return act, y.view(T, self.topk, self.H), shared

    def forward(self, h: torch.Tensor, r: torch.Tensor) -> BlockFP4Outputs:
        """h, r [T, H] bf16. Allocates through torch's caching allocator and never synchronises, so
        it can be recorded in a CUDA graph."""
        self._check(h, r)
        with torch.cuda.device(self.device):
            return self._forward(h, r)

    def _forward(self, h, r) -> BlockFP4Outputs:
        T = h.shape[0]
        normed = self.post_gamma is not None or self.next_gamma is not None or self.residual_scale != 1.0
        x = self._empty(T, self.H) if self.next_gamma is not None else None
        if T == 0:
            e = self._empty(0, self.H)
            return BlockFP4Outputs(e, x, e, self._empty(0, self.topk, dtype=torch.float32),
                                   self._empty(0, self.topk, dtype=torch.int32))
        h1, x2, topw, topi, layout, bn = self._route(h, r)
        _, y, shared = self._experts(x2, topi, layout, bn)
        out = self._empty(T, self.H)
        ops.merge(y, topw, None if normed else h1, shared, out, round_mid=False)
        if normed:
            ops.norm_gate_residual(out, h1, out, x, post_w=self.post_gamma, pre_w=self.next_gamma,
                                   alpha=self.residual_scale, eps=self.eps)
        return BlockFP4Outputs(out, x, h1, topw, topi)

    __call__ = forward

    def calibrate(self, h: torch.Tensor, r: torch.Tensor) -> None:
        """Sets the factors of x2 and of the activations ("nv"; the routed experts' and the shared
        one's have the same) from a batch: their largest magnitudes over 448 * 6, in place, so
        captured graphs use them too."""
        self._check(h, r)
        if self.fmt != "nv" or h.shape[0] == 0:
            return
        with torch.cuda.device(self.device):
            self._calibrate(h, r)

    def _calibrate(self, h, r) -> None:
        h1, x2, topw, topi, layout, bn = self._route(h, r)
        self.x_scales[0].copy_(x2.abs().amax().float().clamp_min(1e-20) / 2688.0)
        act, _, _ = self._experts(x2, topi, layout, bn)
        p = layout[0]
        live = (p < topi.numel()) & (torch.arange(p.numel(), device=p.device) < layout[2])
        top = torch.where(live[:, None], act.abs(), 0.0).amax().float()
        if self.w13s is not None:
            act_s = self._empty(h.shape[0], self.I)
            self.w13s(x2, act_s)
            top = torch.maximum(top, act_s.abs().amax().float())
        self.x_scales[1].copy_(top.clamp_min(1e-20) / 2688.0)
