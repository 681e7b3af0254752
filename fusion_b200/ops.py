"""Torch-tensor wrappers over the C ABI (device pointers + the current CUDA stream).

PyTorch only supplies device memory and streams here; all arithmetic runs in the
library's sm_100a kernels. Every wrapper is destination-passing like the C ABI and
raises ``RuntimeError`` when the library rejects its arguments.
"""

from __future__ import annotations

import ctypes as C

import torch

from . import _lib as L

FUS_EPI_BF16, FUS_EPI_SWIGLU, FUS_EPI_F32 = 0, 1, 2
GEMM_OUT_F32, GEMM_SWIGLU_EXACT, GEMM_W_STREAM, GEMM_MERGE, GEMM_NO_PERSIST = 0x1, 0x2, 0x4, 0x8, 0x10
GEMM_NO_PAIR = 0x40
GEMM_PAIR_NARROW = 0x80
GEMM_SCALE_TOKEN = 0x20
ERR_TIMEOUT, ERR_BAD_EXPERT, ERR_CAPACITY = 0x1, 0x2, 0x4

_status: dict[int, torch.Tensor] = {}


_empty_anchor: dict[int, torch.Tensor] = {}


def _p(t: torch.Tensor | None) -> int | None:
    """Device address of `t`. An empty tensor has no storage (address 0); it is passed as
    an aligned dummy address of its device so that a call over zero rows reaches the
    library's empty-size early return instead of its null-pointer check."""
    if t is None:
        return None
    ptr = t.data_ptr()
    if ptr == 0 and t.numel() == 0 and t.is_cuda:
        idx = t.device.index if t.device.index is not None else torch.cuda.current_device()
        a = _empty_anchor.get(idx)
        if a is None:
            a = torch.zeros(256, dtype=torch.uint8, device=t.device)
            _empty_anchor[idx] = a
        return a.data_ptr()
    return ptr


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def status_tensor(device: torch.device | int | None = None) -> torch.Tensor:
    """The per-device int32 status word the kernels OR error bits into."""
    dev = torch.device("cuda", torch.cuda.current_device() if device is None else
                       (device if isinstance(device, int) else device.index or 0))
    t = _status.get(dev.index)
    if t is None:
        # On a stream of its own, finished here: a first call that is being recorded in a graph must
        # not record this too, or every replay would clear the word. (Allocating beside a
        # capture wants this thread's capture mode relaxed, CU_STREAM_CAPTURE_MODE_RELAXED.)
        side = torch.cuda.Stream(dev)
        exchange, mode = C.CDLL("libcuda.so.1").cuThreadExchangeStreamCaptureMode, C.c_int(2)
        exchange(C.byref(mode))
        try:
            with torch.cuda.stream(side):
                t = torch.zeros(1, dtype=torch.int32, device=dev)
            side.synchronize()
        finally:
            exchange(C.byref(mode))
        t = _status.setdefault(dev.index, t)  # another thread's, if it was first
    return t


def _sp() -> int:
    return status_tensor().data_ptr()


def read_status(clear: bool = True) -> int:
    """Synchronise and return (then clear) the device status bits."""
    t = status_tensor()
    v = int(t.item())
    if clear and v:
        t.zero_()
    return v


def check_status() -> None:
    v = read_status()
    if v:
        names = [n for b, n in ((ERR_TIMEOUT, "timeout"), (ERR_BAD_EXPERT, "bad expert id"),
                                (ERR_CAPACITY, "capacity")) if v & b]
        raise RuntimeError(f"device status {v:#x}: {', '.join(names)}")


def _ld(t: torch.Tensor) -> int:
    assert t.dim() >= 2 and t.stride(-1) == 1, "rows must be contiguous"
    return t.stride(-2)


# -------------------------------------------------------------------------------------
def add_rmsnorm(x, res, w, h1, out, eps: float = 1e-5, do_add: bool = True, do_norm: bool = True):
    T, N = x.shape
    L.call("fus_add_rmsnorm", _p(x), _ld(x), _p(res), _ld(res) if res is not None else 0, _p(w),
           _p(h1), _ld(h1) if h1 is not None else 0, _p(out), _ld(out) if out is not None else 0,
           T, N, eps, int(do_add), int(do_norm), _stream(), _sp())


def router_split_weight(wg: torch.Tensor) -> torch.Tensor:
    """fp32 [E, H] -> bf16 planes [E, 3H] (hi | mid | lo)."""
    E, H = wg.shape
    wa = torch.empty(E, 3 * H, dtype=torch.bfloat16, device=wg.device)
    wg = wg.contiguous()  # held until the launch has returned
    L.call("fus_router_split_weight", _p(wg), _p(wa), E, H, _stream())
    return wa


def router_transpose_weight(wgt: torch.Tensor) -> torch.Tensor:
    """bf16 [H, E] -> bf16 [E, H]."""
    H, E = wgt.shape
    wa = torch.empty(E, H, dtype=torch.bfloat16, device=wgt.device)
    wgt = wgt.contiguous()  # held until the launch has returned
    L.call("fus_router_transpose_weight", _p(wgt), _p(wa), H, E, _stream())
    return wa


def router_nsplit(T: int, H: int, E: int, nplanes: int) -> int:
    return int(L.lib().fus_router_nsplit(T, H, E, nplanes))


def router_logits(x2, wa, nplanes: int, partial, nsplit: int):
    T, H = x2.shape
    E = wa.shape[0]
    L.call("fus_router_logits", _p(x2), _ld(x2), _p(wa), nplanes, _p(partial), T, H, E, nsplit,
           _stream(), _sp())


def router_topk(partial, nsplit: int, bias, logits_out, topw, topi, scale: float = 2.5,
                renorm: bool = True, n_group: int = 1, topk_group: int = 1):
    T, topk = topi.shape
    E = partial.shape[-1]
    if n_group == 1:
        L.call("fus_router_topk", _p(partial), nsplit, _p(bias), _p(logits_out), _p(topw),
               _p(topi), T, E, topk, scale, int(renorm), _stream(), _sp())
    else:
        L.call("fus_router_topk_grouped", _p(partial), nsplit, _p(bias), _p(logits_out),
               _p(topw), _p(topi), T, E, topk, n_group, topk_group, scale, int(renorm),
               _stream(), _sp())


def moe_align_workspace(numel: int, E: int) -> int:
    return int(L.lib().fus_moe_align_workspace(numel, E))


ALIGN_BALANCED = 0x1


def moe_align(ids, E: int, block_m: int, sorted_ids, expert_ids, ntp, workspace=None,
              pos_of=None, flags: int = 0):
    """Dispatch layout; with ``pos_of`` also each pair's dispatch position, with
    ``flags=ALIGN_BALANCED`` each expert's pairs spread evenly over its blocks."""
    flat = ids.reshape(-1)
    assert flat.is_contiguous() and flat.dtype == torch.int32
    need = moe_align_workspace(flat.numel(), E)
    if need and (workspace is None or workspace.numel() < need):
        workspace = torch.empty(need, dtype=torch.uint8, device=ids.device)
    if pos_of is None and not flags:
        L.call("fus_moe_align", _p(flat), flat.numel(), E, block_m, _p(sorted_ids),
               sorted_ids.numel(), _p(expert_ids), expert_ids.numel(), _p(ntp),
               _p(workspace) if need else None, need, _stream(), _sp())
    else:
        L.call("fus_moe_align_ex", _p(flat), flat.numel(), E, block_m, _p(sorted_ids),
               sorted_ids.numel(), _p(expert_ids), expert_ids.numel(), _p(ntp), _p(pos_of),
               flags, _p(workspace) if need else None, need, _stream(), _sp())


def route_small(h, r, gamma, wa, nplanes: int, bias, h1, x2, logits, topw, topi, block_m: int,
                sorted_ids, expert_ids, ntp, done, zero=None, eps: float = 1e-5,
                scale: float = 2.5, renorm: bool = True):
    """Decode front end (T <= 16): norm + router + top-k + layout in one launch."""
    T, H = h.shape
    E = logits.shape[1]
    topk = topi.shape[1]
    L.call("fus_moe_route_small", _p(h), _p(r), _p(gamma), eps, _p(wa), nplanes, _p(bias), T, H, E,
           topk, scale, int(renorm), _p(h1), _p(x2), _p(logits), _p(topw), _p(topi), block_m,
           _p(sorted_ids), sorted_ids.numel(), _p(expert_ids), expert_ids.numel(), _p(ntp),
           _p(done), _p(zero), zero.numel() if zero is not None else 0, _stream(), _sp())


def permute_rows(src, sorted_ids, ntp, div: int, num_valid: int, dst, max_rows: int | None = None):
    H = src.shape[1]
    if max_rows is None:
        max_rows = min(dst.shape[0], sorted_ids.numel())
    L.call("fus_permute_rows", _p(src), _ld(src), _p(sorted_ids), _p(ntp), div, num_valid, _p(dst),
           _ld(dst), max_rows, H, _stream(), _sp())


def gemm_group(w, x, out, *, expert_ids=None, ntp=None, max_blocks: int, row_map=None,
               row_limit: int, row_scale=None, x_rows: int | None = None,
               flags: int = 0, live_ids=None, live_limit: int = 0,
               token_div: int = 1, gather_ids=None, gather_div: int = 1,
               res=None) -> L.GemmGroup:
    """Describe one weight stack + token rows for :func:`grouped_gemm`.

    ``w`` is [n_experts, w_rows, K'] (or [w_rows, K'] for one expert) bf16."""
    g = L.GemmGroup()
    g.w = _p(w)
    g.n_experts = w.shape[0] if w.dim() == 3 else 1
    g.x = _p(x)
    g.ldx = _ld(x)
    g.x_rows = x.shape[0] if x_rows is None else x_rows
    g.expert_ids = _p(expert_ids)
    g.ntp = _p(ntp)
    g.max_blocks = max_blocks
    g.out = _p(out)
    g.ldo = _ld(out)
    g.row_map = _p(row_map)
    g.row_limit = row_limit
    g.row_scale = _p(row_scale)
    g.flags = flags
    g.live_ids = _p(live_ids)
    g.live_limit = live_limit
    g.token_div = token_div
    g.gather_ids = _p(gather_ids)
    g.gather_div = gather_div
    g.res = _p(res)
    g.ldr = _ld(res) if res is not None else 0
    return g


def grouped_gemm(groups: list[L.GemmGroup], w_rows: int, K: int, epilogue: int, block_n: int,
                 a_kplanes: int = 1, ksplit: int = 1, split_stride: int = 0,
                 group_blocks: int = 0):
    arr = (L.GemmGroup * len(groups))(*groups)
    L.call("fus_grouped_gemm_ex", arr, len(groups), w_rows, K, a_kplanes, epilogue, block_n,
           ksplit, split_stride, group_blocks, _stream(), _sp())


def gemm_tiles(w_rows: int, epilogue: int, block_n: int) -> int:
    return int(L.lib().fus_grouped_gemm_tiles(w_rows, epilogue, block_n))


def grouped_gemm_merge(groups: list[L.GemmGroup], w_rows: int, K: int, block_n: int, *,
                       counters, y3, w, res, extra, out, parts: int):
    """Down projection with the expert merge fused into its epilogue.
    y3: [T, topk, H] bf16 rows the routed group writes; counters: zeroed int32
    [T * gemm_tiles(w_rows, FUS_EPI_BF16, block_n)] (left zero afterwards)."""
    m = L.MergeSpec()
    m.counters = _p(counters)
    m.parts = parts
    m.y = _p(y3)
    m.ld_t, m.ld_k = y3.stride(0), y3.stride(1)
    m.topk = y3.shape[1]
    m.w = _p(w)
    m.ldw = w.stride(0)
    m.res = _p(res)
    m.ldr = _ld(res) if res is not None else 0
    m.extra = _p(extra)
    m.lde = _ld(extra) if extra is not None else 0
    m.out = _p(out)
    m.ldo = _ld(out)
    arr = (L.GemmGroup * len(groups))(*groups)
    L.call("fus_grouped_gemm_merge", arr, len(groups), w_rows, K, block_n, C.byref(m), _stream(),
           _sp())


def silu_and_mul(x, y):
    M, twoI = x.shape
    L.call("fus_silu_and_mul", _p(x), _ld(x), _p(y), _ld(y), M, twoI // 2, _stream(), _sp())


def merge(y3, w, res, extra, out, round_mid: bool = True):
    """y3: [T, K, H] view (unit stride along H); extra: bf16 or fp32 [T, H]."""
    T, K, H = y3.shape
    L.call("fus_merge", _p(y3), y3.stride(0), y3.stride(1), K, _p(w),
           w.stride(0) if w is not None else 0, _p(res), _ld(res) if res is not None else 0,
           _p(extra), _ld(extra) if extra is not None else 0,
           int(extra is not None and extra.dtype == torch.float32), _p(out), _ld(out), T, H,
           int(round_mid), _stream(), _sp())


def merge_pos(y, pos_of, K: int, w, res, extra, out):
    """merge over rows in dispatch order: row (t, k) = y[pos_of[t*K + k]] (y: [rows, H])."""
    T, H = out.shape
    L.call("fus_merge_pos", _p(y), _ld(y), _p(pos_of), K, _p(w),
           w.stride(0) if w is not None else 0, _p(res), _ld(res) if res is not None else 0,
           _p(extra), _ld(extra) if extra is not None else 0,
           int(extra is not None and extra.dtype == torch.float32), _p(out), _ld(out), T, H,
           _stream(), _sp())


def oproj_resadd(a, w_nk, res, out, fuse: bool = True, workspace=None):
    """out = bf16(a @ w_nk.T + res) (fuse) or bf16(bf16(a @ w_nk.T) + res); w_nk is the
    K-major [N, K] weight."""
    T, K = a.shape
    N = w_nk.shape[0]
    need = int(L.lib().fus_oproj_workspace(T, N, K, int(fuse)))
    if workspace is None or workspace.numel() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=a.device)
    L.call("fus_oproj_resadd", _p(a), _ld(a), _p(w_nk), T, N, K, _p(res),
           _ld(res) if res is not None else 0, _p(out), _ld(out), int(fuse), _p(workspace),
           need, _stream(), _sp())


def row_rstd(x, rstd, eps: float = 1e-5):
    T, N = x.shape
    L.call("fus_row_rstd", _p(x), _ld(x), T, N, eps, _p(rstd), _stream(), _sp())


def fold_weight(src, w, dst, by_row: bool):
    """dst = bf16(src * w) along K: rows of a [K, N] weight (by_row) or the last dim."""
    if not (src.dtype == w.dtype == dst.dtype == torch.bfloat16):
        raise TypeError("fold_weight: bf16 weight, norm weight and output required")
    assert src.is_contiguous() and dst.is_contiguous()
    cols = src.shape[-1]
    rows = src.numel() // cols
    L.call("fus_fold_weight", _p(src), _p(w), _p(dst), rows, cols, int(by_row),
           src.shape[0] if by_row else 1, _stream(), _sp())


def scale_sum_planes(partial, nsplit: int, row_scale, out):
    T, N = out.shape
    L.call("fus_scale_sum_planes", _p(partial), nsplit, T * N, T, N, _p(row_scale), _p(out),
           _ld(out), _stream(), _sp())


def fp8_block_dequant(src, scale, dst, block=(128, 128)):
    """dst (bf16, rows x cols) = fp8 e4m3 src * scale per block (scale [ceil(R/br),
    ceil(C/bc)] fp32)."""
    if src.dtype != torch.float8_e4m3fn or dst.dtype != torch.bfloat16:
        raise TypeError("fp8_block_dequant: e4m3 source and bf16 destination required")
    cols = src.shape[-1]
    rows = src.numel() // cols
    sc = scale.reshape(-1, scale.shape[-1])
    L.call("fus_fp8_block_dequant", _p(src), _p(sc), sc.stride(0), _p(dst), rows, cols,
           block[0], block[1], _stream(), _sp())


# -------------------------------------------------------------------------------------
# operators over tensors of any device: the call runs on that device, on its current stream.
# At a few tokens the host's work is what a call costs: each function tests everything it
# asks of its arguments in one condition, and only a call that fails it goes through the
# checks that say what is wrong.
DT = {torch.bfloat16: 0, torch.float32: 1, torch.float16: 2}  # FUS_DT_*
FP4_FORMATS = {"mx": 0, "nv": 1}  # FUS_FP4_*
FP4_BLOCK = {"mx": 32, "nv": 16}  # elements that share a scale

_I32, _F32, _U8 = torch.int32, torch.float32, torch.uint8
INT_MAX = 0x7FFFFFFF  # row counts and widths are C ints
_fns: dict = {}
_status_ptr: dict[int, int] = {}
_current_device = torch._C._cuda_getDevice
_raw_stream = torch._C._cuda_getCurrentRawStream


def _dtype(t: torch.Tensor, what: str) -> int:
    code = DT.get(t.dtype)
    if code is None:
        raise TypeError(f"{what}: bf16, fp16 or fp32 required, not {t.dtype}")
    return code


def _need(t, dtype, what: str, shape=None) -> None:
    """`t` (may be None) has this element type, this shape and contiguous elements."""
    if t is None:
        return
    if t.dtype != dtype:
        raise TypeError(f"{what}: {dtype} required, not {t.dtype}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{what}: shape {tuple(t.shape)}, not {tuple(shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{what}: contiguous elements required")


def _rows2d(t: torch.Tensor, what: str) -> int:
    """Row stride of a [rows, columns] tensor whose rows are contiguous."""
    st = t.stride()
    if len(st) != 2 or (st[1] != 1 and t.shape[1] > 1):
        raise ValueError(f"{what}: two dimensions with contiguous rows required")
    return st[0] if t.shape[0] > 1 else t.shape[1]


def _device_of(t: torch.Tensor, *others) -> int:
    """Index of the CUDA device that holds `t` and the others (None: absent)."""
    dev = t.get_device()
    if dev < 0:
        raise ValueError(f"tensors must be on a CUDA device, not {t.device}")
    for o in others:
        if o is not None and o.get_device() != dev:
            raise ValueError(f"tensors on {t.device} and {o.device}")
    return dev


def _call_on(dev: int, name: str, *args) -> None:
    """The entry point with device `dev` current, on its current stream, with its status word.
    Addresses are integers, 0 for none."""
    if dev != _current_device():
        with torch.cuda.device(dev):
            return _call_on(dev, name, *args)
    fn = _fns.get(name)
    if fn is None:
        fn = _fns[name] = L.packed(name)
    status = _status_ptr.get(dev)
    if status is None:
        status = _status_ptr[dev] = status_tensor(dev).data_ptr()
    rc = fn[0](fn[1](*args, _raw_stream(dev), status))
    if rc != 0:
        raise RuntimeError(f"{name} failed ({rc}): {L.last_error()}")


GATE_ACTS = {"none": 0, "sigmoid": 1, "tanh": 2}
SCORES = {"sigmoid": 0, "softmax": 1}


def norm_gate_residual(y, res, h, x=None, *, post_w=None, pre_w=None, gate=None,
                       gate_act: str = "none", alpha: float = 1.0, eps: float = 1e-5):
    """h = res + alpha * act(gate) * norm(y) * post_w and x = norm(h) * pre_w, RMS norms of
    [T, N] rows (bf16, fp16 or fp32 throughout). post_w None: y unnormalised; x None: h only.
    gate: [T, 1], [1, N] or [N], or [T, N]; gate_act "none", "sigmoid" or "tanh". h may be res
    or y itself, x may be y."""
    shape, dtype, dev = y.shape, y.dtype, y.get_device()
    dt = DT.get(dtype)
    ys, rs, hs = y.stride(), res.stride(), h.stride()
    if (dt is None or dev < 0 or len(shape) != 2 or max(shape) > INT_MAX or ys[1] != 1
            or res.shape != shape or res.dtype is not dtype or rs[1] != 1 or res.get_device() != dev
            or h.shape != shape or h.dtype is not dtype or hs[1] != 1 or h.get_device() != dev):
        _refuse_norm(y, res, h, x, post_w, pre_w, gate)
    T, N = shape
    px = ppre = ppost = pgate = 0
    ldx = ldg = kind = 0
    if x is not None:
        if x.shape != shape or x.dtype is not dtype or x.stride()[1] != 1 or x.get_device() != dev:
            _refuse_norm(y, res, h, x, post_w, pre_w, gate)
        px, ldx = x.data_ptr(), x.stride()[0] if T > 1 else N
    if post_w is not None:
        if (post_w.shape != (N,) or post_w.dtype is not dtype or post_w.get_device() != dev
                or not post_w.is_contiguous()):
            _refuse_norm(y, res, h, x, post_w, pre_w, gate)
        ppost = post_w.data_ptr()
    if pre_w is not None:
        if (pre_w.shape != (N,) or pre_w.dtype is not dtype or pre_w.get_device() != dev
                or not pre_w.is_contiguous()):
            _refuse_norm(y, res, h, x, post_w, pre_w, gate)
        ppre = pre_w.data_ptr()
    if gate is not None:
        if gate.dtype is not dtype or gate.get_device() != dev:
            _refuse_norm(y, res, h, x, post_w, pre_w, gate)
        if gate.dim() == 1:
            gate = gate[None]
        what = "norm_gate_residual: gate"
        if gate.shape == shape:
            kind, ldg = 3, _rows2d(gate, what)
        elif gate.shape == (1, N):
            kind = 2
            _rows2d(gate, what)
        elif gate.shape == (T, 1):
            kind, ldg = 1, gate.stride(0)
        else:
            raise ValueError(f"{what} of shape {tuple(gate.shape)} for {(T, N)}")
        pgate = gate.data_ptr()
    one = T <= 1
    _call_on(dev, "fus_norm_gate_residual", y.data_ptr(), N if one else ys[0], res.data_ptr(),
             N if one else rs[0], ppost, pgate, ldg, kind, GATE_ACTS[gate_act], alpha, h.data_ptr(),
             N if one else hs[0], ppre, px, ldx, T, N, dt, eps)


def _refuse_norm(y, res, h, x, post_w, pre_w, gate) -> None:
    what = "norm_gate_residual"
    _dtype(y, what)
    if max(y.shape, default=0) > INT_MAX:
        raise ValueError(f"{what}: {tuple(y.shape)} is too large")
    for t in (y, res, h, x):
        if t is not None and (t.dtype != y.dtype or t.shape != y.shape):
            raise ValueError(f"{what}: res, h and x must have y's type and shape")
        if t is not None:
            _rows2d(t, what)
    for w in (post_w, pre_w):
        _need(w, y.dtype, f"{what}: weight", (y.shape[1],))
    if gate is not None and gate.dtype != y.dtype:
        raise TypeError(f"{what}: gate must have y's type")
    _device_of(y, res, h, x, post_w, pre_w, gate)


def route_topk(logits, topw, topi, *, score: str = "sigmoid", bias=None, n_group: int = 1,
               topk_group: int = 1, renorm: bool = True, scale: float = 1.0):
    """Experts of each token from router logits [T, E] (bf16, fp16 or fp32): topi [T, k] int32
    and their weights topw [T, k] fp32. score "sigmoid" or "softmax"; bias [E] fp32 counts in the
    choice only (+inf: first, -inf: out, not NaN); n_group / topk_group limit the choice to the best
    groups; renorm divides by the chosen weights' sum. -inf or NaN logits mask experts; slots left
    over get id -1, weight 0."""
    T, E = logits.shape
    k = topi.shape[1] if topi.dim() == 2 else 0
    st, dt, dev = logits.stride(), DT.get(logits.dtype), logits.get_device()
    if (dt is None or dev < 0 or T > INT_MAX or E > INT_MAX or st[1] != 1
            or topi.shape != (T, k) or topi.dtype is not _I32 or topi.get_device() != dev
            or topw.shape != (T, k) or topw.dtype is not _F32 or topw.get_device() != dev
            or not topi.is_contiguous() or not topw.is_contiguous()
            or bias is not None and (bias.shape != (E,) or bias.dtype is not _F32
                                     or bias.get_device() != dev or not bias.is_contiguous())):
        _dtype(logits, "route_topk")
        if max(T, E) > INT_MAX:
            raise ValueError(f"route_topk: {(T, E)} is too large")
        _rows2d(logits, "route_topk: logits")
        _need(topi, _I32, "route_topk: topi", (T, k))
        _need(topw, _F32, "route_topk: topw", (T, k))
        _need(bias, _F32, "route_topk: bias", (E,))
        _device_of(logits, topw, topi, bias)
    _call_on(dev, "fus_route_topk", logits.data_ptr(), dt, st[0] if T > 1 else E,
             0 if bias is None else bias.data_ptr(), SCORES[score], n_group, topk_group,
             topw.data_ptr(), topi.data_ptr(), T, E, k, scale, renorm)


def clear_holes(y, ids):
    """Zeros in the rows of y [n, H] (bf16) whose id (int32, n of them) is negative: slots that
    ``route_topk`` left without an expert, which no product writes."""
    if y.dtype != torch.bfloat16:
        raise TypeError("clear_holes: bf16 rows required")
    ldy = _rows2d(y, "clear_holes: y")
    if ids.numel() != y.shape[0]:
        raise ValueError(f"clear_holes: {ids.numel()} ids for {y.shape[0]} rows")
    _need(ids, torch.int32, "clear_holes: ids")
    dev = _device_of(y, ids)
    with torch.cuda.device(dev):
        L.call("fus_clear_holes", _p(ids), ids.numel(), _p(y), ldy, y.shape[1], _stream())


def fp4_scale_bytes(rows: int, K: int, fmt: str, tile: int = 128) -> int:
    """Bytes of the scales of `rows` rows; ``tile`` is the dispatch block of a product's rows
    (or 0: row-major)."""
    n = FP4_BLOCK[fmt]
    if K <= 0 or K % 32 or rows < 0 or tile not in (0, 16, 32, 64, 128, 256):
        raise ValueError(f"fp4_scale_bytes: K={K} (multiples of 32) or tile={tile} not possible")
    if tile == 0:
        return rows * (K // n)
    # whole 512-byte atoms of 128 rows x 4 scales, 256 elements of K at a time
    return -(-rows // tile) * -(-K // 256) * (64 // n) * (tile // 128 or 1) * 512


def _refuse_fp4(values, q, sf, rows: int, K: int, fmt: str, tile: int, gscale, ids, ntp,
                what: str) -> None:
    _dtype(values, what)
    if max(rows, *values.shape) > INT_MAX:
        raise ValueError(f"{what}: {tuple(values.shape)} is too large")
    _rows2d(values, what)
    if fmt not in FP4_FORMATS:
        raise ValueError(f"{what}: format {fmt!r} not in {sorted(FP4_FORMATS)}")
    if q.dtype != _U8 or sf.dtype != _U8:
        raise TypeError(f"{what}: packed values and scales are uint8")
    if q.shape != (rows, K // 2):
        raise ValueError(f"{what}: packed values of shape {tuple(q.shape)}, not {(rows, K // 2)}")
    _rows2d(q, what)
    need = fp4_scale_bytes(rows, K, fmt, tile)
    if not sf.is_contiguous() or sf.numel() < need:
        raise ValueError(f"{what}: scales need {need} contiguous bytes")
    _need(gscale, _F32, what)
    if ids is not None:
        _need(ids, _I32, f"{what}: ids", (rows,))
    _need(ntp, _I32, f"{what}: ntp")
    if ntp is not None and ntp.numel() < 1:
        raise ValueError(f"{what}: ntp is empty")
    _device_of(values, q, sf, gscale, ids, ntp)


def _factors(gscale, rows: int, dev: int, what: str) -> tuple:
    """Address of the factors and rows that share one (0: all)."""
    if gscale.dtype is not _F32 or gscale.get_device() != dev or not gscale.is_contiguous():
        _need(gscale, _F32, what)
        raise ValueError(f"{what}: factors on another device")
    n = gscale.numel()
    if n < 1 or rows % n:
        raise ValueError(f"{what}: {n} factors for {rows} rows")
    return gscale.data_ptr(), rows // n if n > 1 else 0


def fp4_quantize(x, q, sf, fmt: str, *, tile: int = 128, gscale=None, ids=None, id_div: int = 1,
                 id_limit: int = 0, ntp=None):
    """Rows of x [R, K] (bf16, fp16 or fp32) to 4 bits: q [rows, K/2] uint8, sf their scales
    (``fp4_scale_bytes``). ``fmt`` "mx" or "nv"; gscale (nv): fp32 factors, one or one for each
    equal run of rows. With ``ids`` (int32, one for each row of q) row p is x[ids[p] // id_div];
    rows whose id is not in [0, id_limit) keep what they held, as do rows from ntp[0] on."""
    R, K = x.shape
    rows = q.shape[0]
    xs, qs, dt, dev = x.stride(), q.stride(), DT.get(x.dtype), x.get_device()
    if (dt is None or dev < 0 or max(R, K, rows) > INT_MAX or xs[1] != 1 or fmt not in FP4_FORMATS
            or q.shape != (rows, K // 2) or qs[1] != 1 or q.dtype is not _U8 or q.get_device() != dev
            or sf.dtype is not _U8 or sf.get_device() != dev or not sf.is_contiguous()
            or sf.numel() < fp4_scale_bytes(rows, K, fmt, tile)
            or ids is not None and (ids.dtype is not _I32 or ids.shape != (rows,)
                                    or ids.get_device() != dev or not ids.is_contiguous())
            or ntp is not None and (ntp.dtype is not _I32 or ntp.get_device() != dev
                                    or ntp.numel() < 1)):
        _refuse_fp4(x, q, sf, rows, K, fmt, tile, gscale, ids, ntp, "fp4_quantize")
    g, per = (0, 0) if gscale is None else _factors(gscale, rows, dev, "fp4_quantize")
    _call_on(dev, "fus_fp4_quantize", x.data_ptr(), dt, xs[0] if R > 1 else K, R, K,
             FP4_FORMATS[fmt], g, per, 0 if ids is None else ids.data_ptr(), id_div,
             min(id_limit, INT_MAX),
             0 if ntp is None else ntp.data_ptr(), rows, tile, q.data_ptr(),
             qs[0] if rows > 1 else K // 2, sf.data_ptr())


def fp4_dequantize(q, sf, out, fmt: str, *, tile: int = 128, gscale=None):
    """The values of packed rows: out [rows, K] (bf16, fp16 or fp32) = q * scale (* factor)."""
    rows, K = out.shape
    os, qs, dt, dev = out.stride(), q.stride(), DT.get(out.dtype), out.get_device()
    if (dt is None or dev < 0 or max(rows, K) > INT_MAX or os[1] != 1 or fmt not in FP4_FORMATS
            or q.shape != (rows, K // 2) or qs[1] != 1 or q.dtype is not _U8 or q.get_device() != dev
            or sf.dtype is not _U8 or sf.get_device() != dev or not sf.is_contiguous()
            or sf.numel() < fp4_scale_bytes(rows, K, fmt, tile)):
        _refuse_fp4(out, q, sf, rows, K, fmt, tile, gscale, None, None, "fp4_dequantize")
    g, per = (0, 0) if gscale is None else _factors(gscale, rows, dev, "fp4_dequantize")
    _call_on(dev, "fus_fp4_dequantize", q.data_ptr(), qs[0] if rows > 1 else K // 2, sf.data_ptr(),
             FP4_FORMATS[fmt], tile, rows, K, g, per, out.data_ptr(), dt, os[0] if rows > 1 else K)


def fp4_pack_scales(scales, fmt: str, gate_up: bool = False) -> torch.Tensor:
    """Row-major scales [E, N, K/n] (or [N, K/n]) of a weight stack, as a checkpoint stores
    them, in the product's weight layout; ``gate_up`` for a w13 stack multiplied with SwiGLU."""
    if fmt not in FP4_FORMATS:
        raise ValueError(f"fp4_pack_scales: format {fmt!r} not in {sorted(FP4_FORMATS)}")
    s = scales if scales.dim() == 3 else scales[None]
    _need(s, torch.uint8, "fp4_pack_scales")
    E, N, n = s.shape
    K = n * FP4_BLOCK[fmt]
    need = int(L.lib().fus_fp4_weight_scale_bytes(FP4_FORMATS[fmt], E, N, K, int(gate_up)))
    sf = torch.empty(need, dtype=torch.uint8, device=s.device)
    if s.device.type != "cuda":
        raise ValueError("fp4_pack_scales: CUDA tensors required")
    with torch.cuda.device(s.device):
        L.call("fus_fp4_pack_scales", _p(s), FP4_FORMATS[fmt], E, N, K, int(gate_up), _p(sf),
               _stream())
    return sf


def add(a, b, o):
    M, N = a.shape
    L.call("fus_add", _p(a), _ld(a), _p(b), _ld(b), _p(o), _ld(o), M, N, _stream(), _sp())


def seed(o, src=None):
    M, N = o.shape
    L.call("fus_seed", _p(o), _ld(o), _p(src), _ld(src) if src is not None else 0, M, N,
           int(src is not None), _stream(), _sp())


# -------------------------------------------------------------------------------------
def ep_plan(topi, E_loc: int, W: int, dest, leid, counts):
    flat = topi.reshape(-1)
    L.call("fus_ep_plan", _p(flat), flat.numel(), E_loc, W, _p(dest), _p(leid), _p(counts),
           _stream(), _sp())


def ep_dispatch_small(x, topi, E_loc: int, W: int, S: int, rows, leid_out, slot_of_pair):
    T, K = topi.shape
    L.call("fus_ep_dispatch_small", _p(x), _ld(x), x.shape[1], _p(topi), T, K, E_loc, W, S,
           _p(rows), _ld(rows), _p(leid_out), _p(slot_of_pair), _stream(), _sp())


def ep_pack(x, send_ids, n: int, div: int, leid, rows, leid_out):
    L.call("fus_ep_pack", _p(x), _ld(x), x.shape[1], _p(send_ids), n, div, _p(leid), _p(rows),
           _ld(rows), _p(leid_out), _stream(), _sp())


def ep_unpack(rows, send_ids, n: int, y):
    L.call("fus_ep_unpack", _p(rows), _ld(rows), rows.shape[1], _p(send_ids), n, _p(y), _ld(y),
           _stream(), _sp())


def ep_plan_dedup(topi, E_loc: int, W: int, keys, counts):
    """keys[t*W + d] = d if token t has an expert on rank d else -1; counts[d] = rows and
    counts[W + d] = (token, slot) pairs for rank d."""
    T, K = topi.shape
    L.call("fus_ep_plan_dedup", _p(topi), T, K, E_loc, W, _p(keys), _p(counts), _stream(), _sp())


def ep_pack_dedup(x, send_ids, n: int, W: int, topi, topw, E_loc: int, rows, leid_out,
                  pair_pos=None, counts=None, ret_out=None, w_out=None, pos=None,
                  zero_row: int = 0):
    """One row per (token, destination) with its K slots' local expert (-1 off that
    destination); with ret_out, each slot's place in the owner's return rows; with w_out /
    pos, the partial-sum combine's slot weights and merge positions."""
    K = topi.shape[1]
    L.call("fus_ep_pack_dedup", _p(x), _ld(x), x.shape[1], _p(send_ids), n, W, _p(topi),
           _p(topw), K, E_loc, _p(pair_pos), _p(counts), _p(rows), _ld(rows), _p(leid_out),
           _p(ret_out), _p(w_out), _p(pos), zero_row, _stream(), _sp())


def ep_return_rowmap(sorted_ids, ret_idx, K: int, row_prefix, pair_prefix, rowmap, ntp=None):
    """Owner's w2 row map into the return buffer (see fus_ep_return_rowmap); ``ntp``: the
    layout's padded total (entries of sorted_ids past it are not read)."""
    n = ret_idx.numel() // K
    W = row_prefix.numel() - 1
    L.call("fus_ep_return_rowmap", _p(sorted_ids), sorted_ids.numel(), _p(ntp), _p(ret_idx), n, K,
           _p(row_prefix), _p(pair_prefix), W, _p(rowmap), _stream(), _sp())


def ep_partial_sum(y, leid, w, out):
    """out[i] = bf16(sum_j w[i, j] * y[i*K + j] over slots with leid[i, j] >= 0)."""
    n, K = leid.shape
    L.call("fus_ep_partial_sum", _p(y), _ld(y), y.shape[1], _p(leid), _p(w), n, K, _p(out),
           _ld(out), _stream(), _sp())


# -------------------------------------------------------------------------------------
# NVLink peer-memory exchange (CUDA IPC)
def ipc_handle(t: torch.Tensor) -> tuple[bytes, int]:
    """CUDA IPC handle (64 bytes) of the allocation holding ``t`` and t's offset in it."""
    h = (C.c_char * 64)()
    off = C.c_size_t(0)
    L.call("fus_ipc_handle", _p(t), C.cast(h, C.c_void_p), C.byref(off))
    return bytes(h), int(off.value)


def ipc_open(handle: bytes, offset: int) -> int:
    """Map a peer's exported allocation; returns the device address of its offset."""
    h = (C.c_char * 64).from_buffer_copy(handle)
    ptr = C.c_void_p(0)
    L.call("fus_ipc_open", C.cast(h, C.c_void_p), offset, C.byref(ptr))
    return int(ptr.value)


def ipc_close(ptr: int, offset: int):
    L.call("fus_ipc_close", ptr, offset)


def ep_p2p_dispatch(x, topi, E_loc: int, W: int, S: int, rank: int, peer_rows, peer_leid,
                    peer_flags, epoch, slot_of_pair):
    T, K = topi.shape
    L.call("fus_ep_p2p_dispatch", _p(x), _ld(x), x.shape[1], _p(topi), T, K, E_loc, W, S, rank,
           _p(peer_rows), _p(peer_leid), _p(peer_flags), _p(epoch), _p(slot_of_pair),
           _stream(), _sp())


def ep_p2p_wait(flags, epoch, W: int, timeout_ns: int = 0):
    L.call("fus_ep_p2p_wait", _p(flags), _p(epoch), W, timeout_ns, _stream(), _sp())


def ep_p2p_combine(y, recv_leid, W: int, S: int, rank: int, peer_ret, peer_cflags, epoch):
    L.call("fus_ep_p2p_combine", _p(y), _ld(y), y.shape[1], _p(recv_leid), W, S, rank,
           _p(peer_ret), _p(peer_cflags), _p(epoch), _stream(), _sp())


# -------------------------------------------------------------------------------------
def synth_fill(t: torch.Tensor, seed: int, mean: float = 0.0, std: float = 1.0, offset: int = 0):
    """Fill ``t`` (bf16 or fp32, contiguous) with the seeded synthetic stream."""
    assert t.is_contiguous()
    dtype = {torch.bfloat16: 0, torch.float32: 1}[t.dtype]
    if t.is_cuda:
        L.call("fus_synth_fill", _p(t), dtype, t.numel(), offset, seed, mean, std, _stream())
    else:
        L.lib().fus_synth_fill_host(C.c_void_p(t.data_ptr()), dtype, t.numel(), offset, seed,
                                    mean, std)
    return t
