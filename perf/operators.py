"""The 8-bit linear operators around the attention layer, as cases to time.

A layer with 8-bit weights calls them in this order: the norm in front of a
projection with the residual's addition, written as codes and scales
(``norm``); the product of int8 codes with int8 weights under a scale per
token and per channel (``mm``); the gated activation of a feed-forward block,
written as codes and scales (``silu``).  int8 codes have one scale per token
(for the int8 product), e4m3fn codes one per 128 columns (for the block-FP8
product).

``listed`` gives the cases, ``draw`` more of the same ranges, ``prepare`` what
an engine holds before the call, ``run`` one call - through the package's
public functions where ``own`` is true, in elementary torch operations where
it is not - and ``exact`` the same outputs in 64 bits.

Codes are whole numbers that the definition determines: the quotient that is
rounded is formed in 64 bits in the plain form too, so that a value beside a
rounding border falls on the right side of it.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
EPS = 1e-6
GROUP = 128  # columns under one scale of e4m3fn codes
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}


# ------------------------------------------------------------------- cases ----

def listed():
    return [
        # the norm of one decoded token in front of an int8 projection: a launch's latency
        {"name": "norm_decode_1", "op": "norm", "rows": 1, "cols": 7168, "codes": "int8", "type": "bf16",
         "weight": "bf16", "residual": True, "pad": 0},
        # an odd chunk of a prefill in front of a block-FP8 projection, norm weights kept in float32
        {"name": "norm_chunk_2047", "op": "norm", "rows": 2047, "cols": 4096, "codes": "fp8", "type": "bf16",
         "weight": "f32", "residual": True, "pad": 0},
        # rows of an odd width out of a wider buffer, no residual (the first layer's norm)
        {"name": "norm_odd_333", "op": "norm", "rows": 333, "cols": 1501, "codes": "int8", "type": "fp16",
         "weight": "fp16", "residual": False, "pad": 35},
        # a full prefill chunk: the norm of every layer, bound by memory
        {"name": "norm_prefill_8192", "op": "norm", "rows": 8192, "cols": 7168, "codes": "int8", "type": "bf16",
         "weight": "bf16", "residual": True, "pad": 0},
        # the activation between the products of a gated block for a decode step of 8 sequences
        {"name": "silu_decode_8", "op": "silu", "rows": 8, "cols": 2048, "codes": "int8", "type": "bf16"},
        # an odd chunk with codes for the block-FP8 product
        {"name": "silu_chunk_1021", "op": "silu", "rows": 1021, "cols": 4096, "codes": "fp8", "type": "fp16"},
        # a full prefill chunk of a wide block
        {"name": "silu_prefill_8192", "op": "silu", "rows": 8192, "cols": 16384, "codes": "int8", "type": "bf16"},
        # one decoded token against a square projection: the weights stream from memory
        {"name": "mm_decode_1", "op": "mm", "rows": 1, "cols": 7168, "sum": 7168, "out": "bf16", "bias": False},
        # a decode batch of 24 through the low-rank q and kv projection (1536 + 512 channels): few columns, a long sum
        {"name": "mm_decode_24", "op": "mm", "rows": 24, "cols": 2048, "sum": 7168, "out": "bf16", "bias": False},
        # a batch between decode and prefill, with a bias
        {"name": "mm_batch_200", "op": "mm", "rows": 200, "cols": 7168, "sum": 2048, "out": "fp16", "bias": True},
        # odd sizes all round (rows that start at any byte), float32 out
        {"name": "mm_odd_1021", "op": "mm", "rows": 1021, "cols": 4099, "sum": 4111, "out": "f32", "bias": True},
        # a full prefill chunk: bound by the matrix instructions
        {"name": "mm_prefill_8192", "op": "mm", "rows": 8192, "cols": 7168, "sum": 7168, "out": "bf16", "bias": False},
    ]


def _size(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], spread over its logarithm."""
    n = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(n / step)) * step))


def _drawn(rng):
    op = rng.choice(("norm", "norm", "silu", "mm", "mm", "mm"))
    rows = _size(rng, 1, 8192)
    kind = rng.choice(("bf16", "bf16", "fp16"))
    codes = rng.choice(("int8", "int8", "fp8"))
    step = GROUP if codes == "fp8" else rng.choice((1, 8, 8))
    if op == "norm":
        return {"op": op, "rows": rows, "cols": _size(rng, 256, 16384, step), "codes": codes, "type": kind,
                "weight": rng.choice((kind, "f32")), "residual": rng.random() < 0.7,
                "pad": rng.choice((0, 0, 0, 8, 24, 7))}
    if op == "silu":
        return {"op": op, "rows": rows, "cols": _size(rng, 256, 16384, step), "codes": codes, "type": kind}
    step = rng.choice((1, 16, 16, 64))
    return {"op": op, "rows": rows, "cols": _size(rng, 128, 16384, step), "sum": _size(rng, 128, 16384, step),
            "out": rng.choice(("bf16", "bf16", "fp16", "f32")), "bias": rng.random() < 0.4}


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 4e12, w["flops"] / 1e15)


def draw(rng):
    most = {op: max(_cost(c) for c in listed() if c["op"] == op) for op in ("norm", "silu", "mm")}
    while True:
        case = _drawn(rng)
        if _cost(case) <= most[case["op"]]:
            return case


def work(case):
    m, n = case["rows"], case["cols"]
    if case["op"] == "mm":
        k, size = case["sum"], 4 if case["out"] == "f32" else 2
        return {"bytes": m * k + n * k + size * m * n + 4 * (m + n) + (4 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    scales = 4 * m * (n // GROUP if case["codes"] == "fp8" else 1)
    if case["op"] == "silu":
        return {"bytes": 5 * m * n + scales, "flops": 15 * m * n}
    # x and the codes; with a residual also that and the sum that becomes the next one
    each = 7 if case["residual"] else 3
    return {"bytes": each * m * n + scales + n * (4 if case["weight"] == "f32" else 2), "flops": 8 * m * n}


# ------------------------------------------------------------------ inputs ----

def _hidden(g, rows, cols, kind, pad=0):
    """Hidden states: normal values, a few channels many times larger, as in the residual stream of a trained model."""
    x = torch.randn(rows, cols + pad, generator=g, device=DEV)
    loud = torch.randint(0, cols, (max(1, cols // 512),), generator=g, device=DEV)
    x[:, loud] *= 20.0
    return x.to(TYPES[kind])[:, :cols]


def _int8_rows(g, rows, cols):
    """Codes and scales of normal rows: each row's largest value stands at 127."""
    v = torch.randn(rows, cols, generator=g, device=DEV)
    most = v.abs().amax(dim=1, keepdim=True)
    scale = most / 127 * (0.5 + torch.rand(rows, 1, generator=g, device=DEV))
    return torch.round(v * (127 / most)).to(torch.int8), scale


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    m, n = case["rows"], case["cols"]
    s = {"case": case}
    if case["op"] == "norm":
        s["x"] = _hidden(g, m, n, case["type"], case["pad"])
        s["residual"] = _hidden(g, m, n, case["type"]) * 2 if case["residual"] else None
        s["weight"] = (1 + 0.2 * torch.randn(n, generator=g, device=DEV)).to(TYPES[case["weight"]])
    elif case["op"] == "silu":
        # gates mostly negative, as after training
        s["x"] = torch.cat([torch.randn(m, n, generator=g, device=DEV) * 2 - 1,
                            torch.randn(m, n, generator=g, device=DEV)], dim=1).to(TYPES[case["type"]])
    else:
        s["a"], s["scale_a"] = _int8_rows(g, m, case["sum"])
        s["b"], s["scale_b"] = _int8_rows(g, n, case["sum"])
        s["scale_b"] = s["scale_b"] * 0.02
        s["bias"] = torch.randn(n, generator=g, device=DEV) if case["bias"] else None
    return s


# -------------------------------------------------------------- plain forms ----

def _quantise(y, codes):
    """Codes of the 64-bit rows y and the largest magnitude under each scale, in units that a row's common factor leaves open."""
    if codes == "int8":
        most = y.abs().amax(dim=1, keepdim=True)
        return torch.round(y * 127 / torch.where(most > 0, most, 1)).to(torch.int8), most
    z = y.unflatten(1, (-1, GROUP))
    most = z.abs().amax(dim=2, keepdim=True)
    return (z * 448 / torch.where(most > 0, most, 1)).float().to(torch.float8_e4m3fn).flatten(1), most.squeeze(2)


def _plain_norm(s):
    case, x = s["case"], s["x"]
    h = x if s["residual"] is None else (x.float() + s["residual"].float()).to(x.dtype)
    r = torch.rsqrt(h.float().square().mean(dim=1, keepdim=True) + EPS)
    # a row's factor r moves no code: they are the quotients of h w
    codes, most = _quantise(h.double() * s["weight"].double(), case["codes"])
    out = {"codes": codes, "scales": most.float() * r / (127 if case["codes"] == "int8" else 448)}
    return out if s["residual"] is None else {**out, "hidden": h}


def _plain_silu(s):
    gate, up = s["x"].double().chunk(2, dim=1)  # 64 bits: the codes beside a border
    codes, most = _quantise(gate / (1 + torch.exp(-gate)) * up, s["case"]["codes"])
    return {"codes": codes, "scales": most.float() / (127 if s["case"]["codes"] == "int8" else 448)}


def _plain_mm(s):
    out = (s["a"].float() @ s["b"].float().t()) * s["scale_a"] * s["scale_b"].view(1, -1)
    if s["bias"] is not None:
        out = out + s["bias"]
    return out.to(TYPES[s["case"]["out"]])


# ----------------------------------------------------------- this package ----

def _package():
    if "flaggems_vllm" not in sys.modules:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                        "flaggems-vllm_amd"))
    import flaggems_vllm

    return flaggems_vllm


def _own(s):
    fv, case = _package(), s["case"]
    if case["op"] == "mm":
        return fv.int8_scaled_mm(s["a"], s["b"], s["scale_a"], s["scale_b"], s["bias"], TYPES[case["out"]])
    dtype = torch.int8 if case["codes"] == "int8" else torch.float8_e4m3fn
    if case["op"] == "silu":
        codes, scales = fv.fused_silu_mul_quant(s["x"], dtype)
        return {"codes": codes, "scales": scales}
    codes, scales, hidden = fv.fused_add_rms_norm_quant(s["x"], s["residual"], s["weight"], EPS, dtype)
    out = {"codes": codes, "scales": scales}
    return out if s["residual"] is None else {**out, "hidden": hidden}


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    return _plain_norm(state) if op == "norm" else _plain_silu(state) if op == "silu" else _plain_mm(state)


# --------------------------------------------------------------- in 64 bits ----

def _e4m3(v):
    """The e4m3 value nearest to each 64-bit v of at most 448, ties to the even code: steps of 2^(e - 3) in [2^e, 2^(e + 1)), 2^-9 below 2^-6."""
    step = torch.exp2((torch.frexp(v)[1] - 1).clamp(min=-6).double() - 3)
    return torch.round(v / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "mm":
        total = torch.mm(s["a"].double(), s["b"].double().t().contiguous())
        total = total * s["scale_a"].double() * s["scale_b"].double().reshape(-1)
        return total if s["bias"] is None else total + s["bias"].double()
    x = s["x"].double()
    if case["op"] == "silu":
        gate, up = x[:, :case["cols"]], x[:, case["cols"]:]
        y, r, more = up * gate * torch.sigmoid(gate), 1.0, {}
    else:
        h = x
        if s["residual"] is not None:
            h = (x + s["residual"].double()).to(s["x"].dtype).double()
        # y without the row's factor r, an exact product
        y, r = h * s["weight"].double(), 1 / torch.sqrt((h * h).sum(dim=1, keepdim=True) / case["cols"] + EPS)
        more = {} if s["residual"] is None else {"hidden": h}
    if case["codes"] == "int8":
        most = y.abs().max(dim=1, keepdim=True).values
        return {"codes": torch.round(127 * y / most).to(torch.int64), "scales": most * r / 127, **more}
    blocks = y.reshape(case["rows"], -1, GROUP)
    most = blocks.abs().max(dim=2, keepdim=True).values
    return {"codes": _e4m3(448 * blocks / most).reshape(y.shape), "scales": most.squeeze(2) * r / 448, **more}
