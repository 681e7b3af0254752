"""Expert products with 4-bit weights: a weight stack, laid out once, and its call.

``ExpertGemmFP4`` is the 4-bit form of one expert projection (w13 with SwiGLU, or w2): it
quantises bf16 token rows in dispatch order and multiplies them with the packed weights of
each block's expert (``fus_fp4_expert_gemm``: two overlapping launches, no host
synchronisation, graph-capturable). Formats "mx" (32 elements share a power of two) and "nv"
(16 share an e4m3, with one fp32 factor for each expert).
"""

from __future__ import annotations

import ctypes as C

import torch

from . import _lib as L
from . import ops

_OUT = {torch.bfloat16: 0, torch.float32: 1}  # FUS_DT_* of an output


def quantize_weight(w: torch.Tensor, fmt: str):
    """A bf16 / fp16 / fp32 weight stack [E, N, K] in 4 bits, as a checkpoint would hold it:
    packed codes [E, N, K/2] uint8, row-major scale bytes [E, N, K/n] uint8 and, for "nv", the
    experts' fp32 factors [E] (the largest magnitude over 448 * 6), else None."""
    E, N, K = w.shape
    q = torch.empty(E, N, K // 2, dtype=torch.uint8, device=w.device)
    s = torch.empty(E, N, K // ops.FP4_BLOCK[fmt], dtype=torch.uint8, device=w.device)
    g = torch.empty(E, dtype=torch.float32, device=w.device) if fmt == "nv" else None
    for e in range(E):  # one expert at a time: no stack-sized temporary
        if g is not None:
            top = w[e].abs().amax().float() / (448.0 * 6.0)
            g[e] = torch.where(top > 0, top, 1.0)
        ops.fp4_quantize(w[e], q[e], s[e].view(-1), fmt, tile=0,
                         gscale=g[e : e + 1] if g is not None else None)
    return q, s, g


class ExpertGemmFP4:
    """Weights of one projection of E experts: q [E, N, K/2] packed codes and scales
    [E, N, K/n] bytes as ``quantize_weight`` or a checkpoint gives them; ``gscale`` [E] and
    ``x_gscale`` [1] fp32 factors of the weights and the token rows ("nv"; None: 1).
    ``gate_up``: rows [0, N/2) gate, [N/2, N) up, SwiGLU in the epilogue, N/2 outputs."""

    def __init__(self, q: torch.Tensor, scales: torch.Tensor, fmt: str, gscale=None,
                 x_gscale=None, gate_up: bool = False):
        if fmt not in ops.FP4_FORMATS:
            raise ValueError(f"format {fmt!r} not in {sorted(ops.FP4_FORMATS)}")
        if q.dim() != 3:
            raise ValueError("packed weights are [E, N, K/2]")
        ops._need(q, torch.uint8, "packed weights")
        E, N, K = q.shape[0], q.shape[1], q.shape[2] * 2
        if K % 32 or N % 16:
            raise ValueError(f"K={K} must be a multiple of 32 and N={N} of 16")
        ops._need(scales, torch.uint8, "scales", (E, N, K // ops.FP4_BLOCK[fmt]))
        if fmt == "mx":
            gscale = x_gscale = None
        ops._need(gscale, torch.float32, "gscale", (E,))
        ops._need(x_gscale, torch.float32, "x_gscale")
        if x_gscale is not None and x_gscale.numel() != 1:
            raise ValueError("x_gscale: one factor")
        self._dev = ops._device_of(q, scales, gscale, x_gscale)
        self.E, self.N, self.K, self.fmt, self.gate_up = E, N, K, fmt, gate_up
        self.cols = N // 2 if gate_up else N
        self.device = q.device
        self._keep = (q, ops.fp4_pack_scales(scales, fmt, gate_up), gscale, x_gscale)
        d = L.Fp4GemmDesc()
        d.wq, d.wsf, d.wg, d.xg = (ops._p(t) for t in self._keep[:3] + (x_gscale,))
        d.n_experts, d.w_rows, d.K, d.fmt = E, N, K, ops.FP4_FORMATS[fmt]
        d.ldxq = -(-K // 32) * 16
        d.epilogue = ops.FUS_EPI_SWIGLU if gate_up else ops.FUS_EPI_BF16
        self._desc = d

    def __call__(self, x, out, sorted_ids=None, expert_ids=None, ntp=None, block_n: int = 0, *,
                 topk: int = 1, gather: bool = True, scatter: bool = True, pairs: int | None = None,
                 row_scale=None):
        """One projection over a dispatch layout (``ops.moe_align`` with block_n: pads end a block, a
        pair stands at most once).

        gather: x [T, K] holds tokens, dispatch row p is x[sorted_ids[p] // topk]; else x
        [capacity, K] is in dispatch order. scatter: out [pairs, cols] in pair order (row
        sorted_ids[p]), else out [capacity, cols] in dispatch order; rows of pads are left as
        they were. pairs: T * topk, needed when neither gather nor scatter tells it. out is bf16
        or fp32; row_scale: fp32, one for each row of out.

        Without sorted_ids the one expert multiplies every row: x [T, K], out [T, cols]."""
        dev = self._dev
        xs, os = x.stride(), out.stride()
        T, rows = x.shape[0], out.shape[0]
        dt, odt = ops.DT.get(x.dtype), _OUT.get(out.dtype)
        if (dt is None or odt is None or x.shape != (T, self.K) or out.shape != (rows, self.cols)
                or xs[1] != 1 or os[1] != 1 or x.get_device() != dev or out.get_device() != dev
                or row_scale is not None and (
                    row_scale.dtype is not torch.float32 or row_scale.numel() < rows
                    or row_scale.get_device() != dev or not row_scale.is_contiguous())):
            self._refuse(x, out, row_scale)
        d = L.Fp4GemmDesc.from_buffer_copy(self._desc)
        spread = 0
        if sorted_ids is None:
            if self.E != 1 or expert_ids is not None or ntp is not None:
                raise ValueError("without sorted_ids: one expert, no expert_ids, no ntp")
            cap = T
            block_n = block_n or dense_block_n(cap)
            gather = scatter = False
            if max(T, rows) > ops.INT_MAX:
                raise ValueError("too many rows")
        else:
            for t in (sorted_ids, expert_ids, ntp):
                if t.dtype is not torch.int32 or t.get_device() != dev or not t.is_contiguous():
                    ops._need(t, torch.int32, "sorted_ids, expert_ids and ntp")
                    raise ValueError(f"tensors must be on {self.device}, with the weights")
            cap = sorted_ids.numel()
            if block_n < 1 or cap % block_n or expert_ids.numel() < cap // block_n or ntp.numel() < 1:
                raise ValueError("sorted_ids must hold whole blocks, expert_ids one id for each, "
                                 "ntp the padded total")
            if topk < 1 or pairs is not None and pairs < 0:
                raise ValueError(f"topk={topk}, pairs={pairs} not possible")
            if gather:
                pairs = T * topk
                spread = 4 * pairs
            elif pairs is None:
                if not scatter:
                    raise ValueError("rows in and out in dispatch order: pairs (T * topk) required")
                pairs = rows
            if max(cap, rows, pairs) > ops.INT_MAX:
                raise ValueError("too many rows")
            if pairs == 0:
                return out
            d.expert_ids, d.ntp = expert_ids.data_ptr(), ntp.data_ptr()
            d.live_ids, d.live_limit, d.scatter = sorted_ids.data_ptr(), pairs, scatter
        if rows < (pairs if scatter else cap) or not gather and T < cap:
            raise ValueError("too few rows")
        # the packed rows: fresh for each call, so calls on other streams and captured graphs
        # never share them; `buf` holds them until the launches have returned (another thread's
        # allocation on this stream would be given their memory before)
        packed = cap * d.ldxq
        size = packed + ops.fp4_scale_bytes(cap, self.K, self.fmt, block_n)
        buf = torch.empty(size + spread, dtype=torch.uint8, device=self.device)
        ws = buf.data_ptr()
        d.xq, d.xsf = ws, ws + packed
        d.x_rows, d.block_n = cap, block_n
        if row_scale is not None:
            d.row_scale = row_scale.data_ptr()
        d.out, d.ldo = out.data_ptr(), os[0] if rows > 1 else self.cols
        d.out_rows, d.out_dtype = rows, odt
        ops._call_on(dev, "fus_fp4_expert_gemm", C.addressof(d), x.data_ptr(), dt,
                     xs[0] if T > 1 else self.K, T, topk if gather else 0,
                     ws + size if spread else 0)
        del buf
        return out

    def _refuse(self, x, out, row_scale) -> None:
        ops._dtype(x, "x")
        if out.dtype not in _OUT:
            raise TypeError("out is bf16 or fp32")
        if x.shape != (len(x), self.K) or out.shape != (len(out), self.cols):
            raise ValueError(f"x [.., {self.K}] and out [.., {self.cols}] required")
        ops._rows2d(x, "x")
        ops._rows2d(out, "out")
        ops._need(row_scale, torch.float32, "row_scale")
        if row_scale is not None and row_scale.numel() < out.shape[0]:
            raise ValueError("row_scale: one for each row of out")
        if ops._device_of(x, out, row_scale) != self._dev:
            raise ValueError(f"tensors must be on {self.device}, with the weights")


def dense_block_n(rows: int) -> int:
    """Token block of a product whose rows all meet one weight: the smallest that holds them,
    256 at most."""
    for bn in (16, 32, 64, 128):
        if rows <= bn:
            return bn
    return 256
