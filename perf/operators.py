"""Cases of the four-bit expert path, the routing and the block norms, for measuring them.

Four operators around the MoE block:

* ``quantize``: rows to microscaled 4-bit floating point and back to the values they stand
  for. ``mx``: 32 elements share a power of two; ``nv``: 16 elements share an e4m3 scale
  times one fp32 factor of the whole tensor.
* ``experts``: the grouped product of quantised token rows with quantised expert weights,
  in dispatch order, optionally with SwiGLU over the gate and up halves.
* ``route``: softmax or sigmoid scores of the experts, a balancing bias in the choice only,
  groups, top-k, renormalised weights.
* ``norms``: the norm after a block, its gate and residual scale, the residual sum, and the
  norm before the next block.

``own`` chooses between the plain form (elementary torch operations) and the framework's
calls; both take what ``prepare`` made.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # the magnitudes of e2m1, by code
BLOCK = {"mx": 32, "nv": 16}  # elements that share a scale


def listed():
    return [
        # one decoded token's routed rows, quantised before the experts
        {"name": "quantize-decode-mx", "op": "quantize", "fmt": "mx", "rows": 8, "K": 6144, "dtype": "bf16"},
        # a prompt's hidden states
        {"name": "quantize-prefill-nv", "op": "quantize", "fmt": "nv", "rows": 8192, "K": 6144, "dtype": "bf16"},
        # fp32 rows of a ragged batch, a length that fills no whole tile
        {"name": "quantize-ragged-mx", "op": "quantize", "fmt": "mx", "rows": 1333, "K": 2080, "dtype": "fp32"},
        # one token through 8 of 256 experts: gate and up projections
        {"name": "experts-decode1-nv", "op": "experts", "fmt": "nv", "T": 1, "E": 256, "topk": 8, "N": 4096, "K": 6144, "swiglu": True},
        # 32 tokens decoded together: down projections, most experts touched
        {"name": "experts-decode32-mx", "op": "experts", "fmt": "mx", "T": 32, "E": 256, "topk": 8, "N": 6144, "K": 2048, "swiglu": False},
        # one of 8 GPUs' 32 experts at a prompt of 8192 tokens: about 256 rows for each expert
        {"name": "experts-prefill-nv", "op": "experts", "fmt": "nv", "T": 1024, "E": 32, "topk": 8, "N": 4096, "K": 6144, "swiglu": True},
        # one decoded token
        {"name": "route-decode", "op": "route", "score": "sigmoid", "bias": True, "T": 1, "E": 256, "topk": 8, "groups": 1, "topk_group": 1, "renorm": True, "scale": 2.5, "dtype": "fp32"},
        # a long prompt, grouped experts
        {"name": "route-prefill-groups", "op": "route", "score": "sigmoid", "bias": True, "T": 32768, "E": 256, "topk": 8, "groups": 8, "topk_group": 4, "renorm": True, "scale": 2.5, "dtype": "fp32"},
        # softmax scores from bf16 logits (many exact ties), an odd count of tokens and experts
        {"name": "route-softmax-ragged", "op": "route", "score": "softmax", "bias": False, "T": 4099, "E": 162, "topk": 6, "groups": 1, "topk_group": 1, "renorm": False, "scale": 1.0, "dtype": "bf16"},
        # one decoded token between two blocks
        {"name": "norms-decode", "op": "norms", "T": 1, "N": 6144, "dtype": "bf16", "gate": "none", "act": "none", "alpha": 1.0},
        # a prompt: gate for each token
        {"name": "norms-prefill", "op": "norms", "T": 8192, "N": 6144, "dtype": "bf16", "gate": "token", "act": "sigmoid", "alpha": 0.5},
        # an odd width, where rows do not start on 16 bytes; gate for each channel
        {"name": "norms-ragged", "op": "norms", "T": 777, "N": 5003, "dtype": "fp16", "gate": "channel", "act": "tanh", "alpha": 0.22},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("quantize", "experts", "route", "norms"))
    if op == "quantize":
        return {"op": op, "fmt": rng.choice(("mx", "nv")), "rows": _log(rng, 1, 8192), "K": 32 * _log(rng, 2, 192), "dtype": rng.choice(("bf16", "fp16", "fp32"))}
    if op == "experts":
        E = _log(rng, 4, 32)
        topk = rng.randint(1, min(E, 8))
        return {"op": op, "fmt": rng.choice(("mx", "nv")), "T": _log(rng, 1, 1024), "E": E, "topk": topk, "N": 16 * _log(rng, 8, 256), "K": 32 * _log(rng, 4, 192), "swiglu": rng.random() < 0.5}
    if op == "route":
        groups = rng.choice((1, 1, 4, 8))
        E = groups * _log(rng, 8, 64) if groups > 1 else _log(rng, 16, 512)
        return {"op": op, "score": rng.choice(("sigmoid", "softmax")), "bias": rng.random() < 0.5, "T": _log(rng, 1, 16384), "E": E, "topk": rng.randint(1, 8), "groups": groups, "topk_group": max(1, groups // 2), "renorm": rng.random() < 0.5, "scale": rng.choice((1.0, 2.5)), "dtype": rng.choice(("fp32", "bf16"))}
    return {"op": op, "T": _log(rng, 1, 8192), "N": _log(rng, 64, 6144), "dtype": rng.choice(("bf16", "fp16")), "gate": rng.choice(("none", "token", "channel", "full")), "act": rng.choice(("none", "sigmoid", "tanh")), "alpha": rng.choice((1.0, 0.5, 0.22))}


def _block_n(rows, E):
    """Token rows for a dispatch block, by the average for an expert."""
    each = rows / E
    return 16 if each <= 12 else 32 if each <= 24 else 64 if each <= 48 else 128 if each <= 96 else 256


# ---- what a user's program has in hand -------------------------------------------------


def _layout(topi, E, bn):
    """Flat (token, slot) ids by expert, each expert's run padded to `bn` with the count of ids."""
    flat = topi.reshape(-1).long()
    R = flat.numel()
    order = torch.argsort(flat, stable=True)
    count = torch.bincount(flat, minlength=E)
    padded = (count + bn - 1) // bn * bn
    start = torch.cumsum(padded, 0) - padded
    first = torch.cumsum(count, 0) - count
    by = flat[order]
    at = start[by] + torch.arange(R, device=flat.device) - first[by]
    total = int(padded.sum())
    sorted_ids = torch.full((total,), R, dtype=torch.int32, device=flat.device)
    sorted_ids[at] = order.int()
    expert_ids = torch.repeat_interleave(torch.arange(E, device=flat.device), padded // bn).int()
    ntp = torch.tensor([total], dtype=torch.int32, device=flat.device)
    return sorted_ids, expert_ids, ntp


def _weights(case, g):
    """Expert weights as a checkpoint holds them: packed codes (the even element in the low
    four bits), scale bytes, and for nv one fp32 factor for each expert."""
    E, N, K, n = case["E"], case["N"], case["K"], BLOCK[case["fmt"]]
    q = torch.empty(E, N, K // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(E, N, K // n, dtype=torch.uint8, device="cuda")
    factor = torch.ones(E, device="cuda")
    step = max(1, (1 << 28) // (N * K))
    for e in range(0, E, step):
        w = torch.randn(min(step, E - e), N, K, device="cuda", generator=g) * 0.02
        if case["fmt"] == "nv":
            factor[e : e + step] = w.abs().amax((1, 2)) / (448.0 * 6.0)
        code, byte = _encode(w, case["fmt"], factor[e : e + step, None, None, None])
        q[e : e + step] = code[..., 0::2] | (code[..., 1::2] << 4)
        scales[e : e + step] = byte
    return q, scales, factor


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op = case["op"]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if op == "quantize":
        # hidden states: most values near one, a few channels far larger
        x = randn(case["rows"], case["K"]) * torch.exp(0.7 * randn(1, case["K"]))
        x = x.to(DTYPES[case["dtype"]])
        factor = (x.float().abs().max() / (448.0 * 6.0)).reshape(1)
        return {"case": case, "x": x, "factor": factor}
    if op == "experts":
        T, E, topk = case["T"], case["E"], case["topk"]
        x = randn(T, case["K"]).to(torch.bfloat16)
        topi = torch.topk(torch.rand(T, E, device="cuda", generator=g), topk, dim=-1).indices.int()
        bn = _block_n(T * topk, E)
        sorted_ids, expert_ids, ntp = _layout(topi, E, bn)
        q, scales, factor = _weights(case, g)
        x_factor = (x.float().abs().max() / (448.0 * 6.0)).reshape(1)
        state = {"case": case, "x": x, "sorted_ids": sorted_ids, "expert_ids": expert_ids, "ntp": ntp, "bn": bn, "x_factor": x_factor}
        if own:
            from fusion_b200.fp4 import ExpertGemmFP4

            state["experts"] = ExpertGemmFP4(q, scales, case["fmt"], gscale=factor, x_gscale=x_factor, gate_up=case["swiglu"])
        else:
            state |= {"q": q, "scales": scales, "factor": factor}
        return state
    if op == "route":
        logits = randn(case["T"], case["E"]).to(DTYPES[case["dtype"]])
        bias = 0.02 * randn(case["E"]) if case["bias"] else None
        return {"case": case, "logits": logits, "bias": bias}
    T, N, dt = case["T"], case["N"], DTYPES[case["dtype"]]
    shape = {"none": None, "token": (T, 1), "channel": (1, N), "full": (T, N)}[case["gate"]]
    return {
        "case": case,
        "y": (2.0 * randn(T, N)).to(dt),
        "res": randn(T, N).to(dt),
        "post_w": (1.0 + 0.02 * randn(N)).to(dt),
        "pre_w": (1.0 + 0.02 * randn(N)).to(dt),
        "gate": randn(*shape).to(dt) if shape else None,
    }


# ---- the plain forms ----------------------------------------------------------------------


def _encode(x, fmt, factor):
    """Codes (0..15) and scale bytes of the blocks along the last axis; `factor` broadcasts
    over [..., blocks, 1]."""
    n = BLOCK[fmt]
    v = x.reshape(*x.shape[:-1], x.shape[-1] // n, n)
    amax = v.abs().amax(-1, keepdim=True)
    if fmt == "mx":
        # the power of two that brings the largest into [4, 8); 6 holds what is over it
        byte = torch.where(amax > 0, torch.frexp(amax)[1] - 3 + 127, 0).clamp(0, 254)
        scale = torch.exp2(byte.to(v.dtype) - 127)
    else:
        # e4m3, to the nearest, ties to even
        t = amax / (6.0 * factor.to(v.dtype))
        exponent = torch.where(t > 0, torch.frexp(t)[1] - 1, -6).clamp(-6, 8)
        mantissa = torch.round(t * torch.exp2((3 - exponent).to(v.dtype)))
        byte = torch.clamp((exponent + 6) * 8 + mantissa.to(exponent.dtype), max=126)
        scale = torch.clamp(mantissa * torch.exp2((exponent - 3).to(v.dtype)), max=448.0) * factor.to(v.dtype)
    a = torch.where(scale > 0, v.abs() / scale, 0.0)
    code = (a > 0.25).to(torch.uint8)
    code += a >= 0.75
    code += a > 1.25
    code += a >= 1.75
    code += a > 2.5
    code += a >= 3.5
    code += a > 5.0
    code |= torch.signbit(v).to(torch.uint8) << 3
    return code.reshape(x.shape), byte.squeeze(-1).to(torch.uint8)


def _decode(code, byte, fmt, factor):
    """The values, fp32, of codes [..., K] and scale bytes [..., K / n]."""
    n = BLOCK[fmt]
    table = torch.tensor(GRID + tuple(-v for v in GRID), device=code.device)
    if fmt == "mx":
        scale = torch.exp2(byte.float() - 127)
    else:
        scale = byte.view(torch.float8_e4m3fn).float()
    v = table[code.int()].reshape(*byte.shape, n) * scale[..., None]
    return (v if fmt == "mx" else v * factor).reshape(code.shape)


def _unpack(q):
    return torch.stack((q & 15, q >> 4), -1).reshape(*q.shape[:-1], 2 * q.shape[-1])


def _rounded(x, fmt, factor):
    """x as 4 bits hold it, in fp32."""
    code, byte = _encode(x.double() if fmt == "nv" else x.float(), fmt, factor)
    return _decode(code, byte, fmt, factor)


def _plain_experts(s):
    c, bn = s["case"], s["bn"]
    R, blocks = c["T"] * c["topk"], s["expert_ids"].numel()
    x = _rounded(s["x"], c["fmt"], s["x_factor"])
    live = s["sorted_ids"] < R
    rows = x[torch.where(live, s["sorted_ids"], 0) // c["topk"]].reshape(blocks, bn, c["K"])
    which = s["expert_ids"]
    w = _decode(_unpack(s["q"][which]), s["scales"][which], c["fmt"], s["factor"][which][:, None, None, None])
    y = torch.bmm(rows, w.transpose(1, 2)).reshape(blocks * bn, c["N"])
    if c["swiglu"]:
        gate, up = y.chunk(2, -1)
        y = gate / (1.0 + torch.exp(-gate)) * up
    out = torch.empty(R, y.shape[1], dtype=torch.bfloat16, device=y.device)
    out[s["sorted_ids"][live].long()] = y[live].to(torch.bfloat16)
    return {"y": out}


def _plain_route(s):
    c = s["case"]
    # 64 bits: a choice between neighbours must not hang on a rounding
    l = s["logits"].double()
    if c["score"] == "sigmoid":
        score = 1.0 / (1.0 + torch.exp(-l))
    else:
        e = torch.exp(l - l.amax(-1, keepdim=True))
        score = e / e.sum(-1, keepdim=True)
    choice = score + s["bias"].double() if s["bias"] is not None else score
    if c["groups"] > 1:
        grouped = choice.reshape(c["T"], c["groups"], -1)
        best = torch.sort(grouped, dim=-1, descending=True).values[..., :2].sum(-1)
        keep = torch.sort(best, dim=-1, descending=True, stable=True).indices[:, : c["topk_group"]]
        mask = torch.zeros(c["T"], c["groups"], dtype=torch.bool, device=l.device).scatter(1, keep, True)
        choice = torch.where(mask[..., None], grouped, -math.inf).reshape(c["T"], -1)
    topi = torch.sort(choice, dim=-1, descending=True, stable=True).indices[:, : c["topk"]]
    w = torch.gather(score, 1, topi)
    if c["renorm"]:
        w = w / w.sum(-1, keepdim=True)
    return {"weights": (w * c["scale"]).float(), "ids": topi.int()}


def _norm(v, w):
    return v * torch.rsqrt((v * v).mean(-1, keepdim=True) + 1e-5) * w.float()


def _plain_norms(s):
    c, dt = s["case"], s["y"].dtype
    v = _norm(s["y"].float(), s["post_w"]) * c["alpha"]
    if s["gate"] is not None:
        gate = s["gate"].float()
        if c["act"] == "sigmoid":
            gate = 1.0 / (1.0 + torch.exp(-gate))
        elif c["act"] == "tanh":
            gate = torch.tanh(gate)
        v = v * gate
    h = s["res"].float() + v
    return {"h": h.to(dt), "x": _norm(h, s["pre_w"]).to(dt)}


def run(state):
    c = state["case"]
    if not own:
        if c["op"] == "quantize":
            return {"values": _rounded(state["x"], c["fmt"], state["factor"]).to(state["x"].dtype)}
        return {"experts": _plain_experts, "route": _plain_route, "norms": _plain_norms}[c["op"]](state)
    from fusion_b200 import ops

    if c["op"] == "quantize":
        x = state["x"]
        factor = state["factor"] if c["fmt"] == "nv" else None
        q = torch.empty(c["rows"], c["K"] // 2, dtype=torch.uint8, device=x.device)
        sf = torch.empty(ops.fp4_scale_bytes(c["rows"], c["K"], c["fmt"]), dtype=torch.uint8, device=x.device)
        ops.fp4_quantize(x, q, sf, c["fmt"], gscale=factor)
        out = torch.empty_like(x)
        ops.fp4_dequantize(q, sf, out, c["fmt"], gscale=factor)
        return {"values": out}
    if c["op"] == "experts":
        x = state["x"]
        cols = c["N"] // 2 if c["swiglu"] else c["N"]
        out = torch.empty(c["T"] * c["topk"], cols, dtype=torch.bfloat16, device=x.device)
        state["experts"](x, out, state["sorted_ids"], state["expert_ids"], state["ntp"], state["bn"], topk=c["topk"])
        return {"y": out}
    if c["op"] == "route":
        logits = state["logits"]
        topw = torch.empty(c["T"], c["topk"], device=logits.device)
        topi = torch.empty(c["T"], c["topk"], dtype=torch.int32, device=logits.device)
        ops.route_topk(logits, topw, topi, score=c["score"], bias=state["bias"], n_group=c["groups"], topk_group=c["topk_group"], renorm=c["renorm"], scale=c["scale"])
        return {"weights": topw, "ids": topi}
    y = state["y"]
    h, x = torch.empty_like(y), torch.empty_like(y)
    ops.norm_gate_residual(y, state["res"], h, x, post_w=state["post_w"], pre_w=state["pre_w"], gate=state["gate"], gate_act=c["act"], alpha=c["alpha"], eps=1e-5)
    return {"h": h, "x": x}


# ---- the cost that no form can do without -----------------------------------------------------


def work(case):
    op = case["op"]
    if op == "quantize":
        n = case["rows"] * case["K"]
        size = 4 if case["dtype"] == "fp32" else 2
        # the rows read, their packed form written and read again, the values written
        return {"bytes": n * (2 * size + 2 * (0.5 + 1 / BLOCK[case["fmt"]])), "flops": 3 * n}
    if op == "experts":
        R, E, N, K = case["T"] * case["topk"], case["E"], case["N"], case["K"]
        touched = E * (1 - (1 - case["topk"] / E) ** case["T"])
        weight = touched * N * K * (0.5 + 1 / BLOCK[case["fmt"]])
        return {"bytes": weight + case["T"] * K * 2 + R * (N // 2 if case["swiglu"] else N) * 2 + 4 * R, "flops": 2.0 * R * N * K}
    if op == "route":
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": case["T"] * (case["E"] * size + case["topk"] * 8), "flops": case["T"] * case["E"] * 6}
    n, size = case["T"] * case["N"], 4 if case["dtype"] == "fp32" else 2
    return {"bytes": n * size * (5 if case["gate"] == "full" else 4), "flops": 10 * n}


# ---- the definitions in 64 bits -----------------------------------------------------------------


def _exact_values(x, fmt, factor):
    """The nearest 4-bit values of x, from the definition, in 64 bits."""
    n = BLOCK[fmt]
    v = x.double().reshape(*x.shape[:-1], -1, n)
    top = v.abs().max(-1, keepdim=True).values
    if fmt == "mx":
        scale = torch.ldexp(torch.ones_like(top), torch.frexp(top.clamp_min(2.0**-125)).exponent - 3)
    else:
        codes = torch.arange(127, dtype=torch.uint8, device=x.device)
        grid = codes.view(torch.float8_e4m3fn).double()
        middle = (grid[1:] + grid[:-1]) / 2
        want = top / (6.0 * factor.double())
        i = torch.searchsorted(middle, want)
        tie = (i < middle.numel()) & (middle[i.clamp_max(middle.numel() - 1)] == want)
        i = torch.where(tie & (i % 2 == 1), i + 1, i)
        scale = grid[i] * factor.double()
    y = torch.where(scale > 0, v / scale, torch.zeros_like(v))
    exponent = torch.floor(torch.log2(y.abs().clamp_min(1.0)))
    step = torch.pow(2.0, exponent - 1)
    y = (torch.round(y / step) * step).clamp(-6.0, 6.0)
    return (y * scale).reshape(x.shape)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    op = case["op"]
    if op == "quantize":
        return {"values": _exact_values(s["x"], case["fmt"], s["factor"])}
    if op == "experts":
        R = case["T"] * case["topk"]
        x = _exact_values(s["x"], case["fmt"], s["x_factor"])
        grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
        out = torch.empty(R, case["N"] // 2 if case["swiglu"] else case["N"], dtype=torch.float64, device=x.device)
        owner = s["expert_ids"].repeat_interleave(s["bn"])
        for e in torch.unique(s["expert_ids"]).tolist():
            ids = s["sorted_ids"][(owner == e) & (s["sorted_ids"] < R)].long()
            byte, packed = s["scales"][e], s["q"][e]
            scale = torch.pow(2.0, byte.double() - 127) if case["fmt"] == "mx" else byte.view(torch.float8_e4m3fn).double() * s["factor"][e].double()
            w = torch.empty(case["N"], case["K"], dtype=torch.float64, device=x.device)
            for half in (0, 1):
                c = (packed >> (4 * half)) & 15
                w[:, half::2] = grid[(c & 7).long()] * (1.0 - 2.0 * (c >> 3).double())
            w = (w.reshape(case["N"], -1, BLOCK[case["fmt"]]) * scale[..., None]).reshape(case["N"], case["K"])
            y = x[ids // case["topk"]] @ w.T
            if case["swiglu"]:
                a, b = y[:, : case["N"] // 2], y[:, case["N"] // 2 :]
                y = a * torch.sigmoid(a) * b
            out[ids] = y
        return {"y": out}
    if op == "route":
        l = s["logits"].double()
        p = torch.sigmoid(l) if case["score"] == "sigmoid" else torch.softmax(l, -1)
        ids = _plain_route(s)["ids"].long()
        w = p.gather(1, ids)
        if case["renorm"]:
            w = w / w.sum(1, keepdim=True)
        return {"weights": w * case["scale"], "ids": None}
    y, res = s["y"].double(), s["res"].double()
    v = y / torch.sqrt(y.square().mean(-1, keepdim=True) + 1e-5) * s["post_w"].double()
    if s["gate"] is not None:
        v = v * {"none": lambda t: t, "sigmoid": torch.sigmoid, "tanh": torch.tanh}[case["act"]](s["gate"].double())
    h = res + case["alpha"] * v
    return {"h": h, "x": h / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-5) * s["pre_w"].double()}
