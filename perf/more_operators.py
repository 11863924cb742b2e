"""The operators of a block served in 8-bit integers, as cases that can be timed.

Three kinds of work, through the public entry points of cublade_amd.quantization:

  linear   linear_w8a8: the product of INT8 activations (one scale for each
           token) and INT8 weights (one scale for each output channel)
  gated    gated_w8a8: the first half of a gated feed-forward block, both
           projections, the activation and the product in one kernel
  norm     norm_tensor and residual_norm: the norms before and after a block,
           with the block's gate and residual scale, whose result leaves as
           INT8 codes with a scale for each token, or in 16 bits

Where ``own`` is false, ``run`` computes the same from elementary torch
operations in 32 bits; ``exact`` gives the result in 64 bits, from the
definition. Codes are returned as the values they stand for (dequantize_tensor).
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"fp16": 2, "bf16": 2, "fp32": 4}
EPS = 1e-12          # of a scale's maximum
NORM_EPS = 1e-6


def listed() -> list[dict]:
    return [
        # One token through a square projection. Latency.
        dict(name="linear_one", kind="linear", m=1, n=4096, k=4096, xmode="token", bias=False,
             dtype="bf16"),
        # A decode step of 16 users through an up projection: the weight's bytes.
        dict(name="linear_decode", kind="linear", m=16, n=11008, k=4096, xmode="token", bias=False,
             dtype="fp16"),
        # A step with drafted tokens, or a short prompt, through the down
        # projection: too many rows to be bound by the weight, few for tiles.
        dict(name="linear_few", kind="linear", m=200, n=4096, k=11008, xmode="token", bias=False,
             dtype="bf16"),
        # An odd layer: rows that are no multiple of 16 bytes, a bias, a static
        # scale of the whole input.
        dict(name="linear_odd", kind="linear", m=333, n=1001, k=1403, xmode="tensor", bias=True,
             dtype="fp16"),
        # A prompt of 4096 tokens through a large model's up projection.
        dict(name="linear_prompt", kind="linear", m=4096, n=28672, k=8192, xmode="token",
             bias=False, dtype="bf16"),
        # One token through a gated block's first half.
        dict(name="gated_one", kind="gated", m=1, n=11008, k=4096, act="silu", bias=False,
             dtype="bf16"),
        # A ragged batch of a small model with GELU gates and biases.
        dict(name="gated_odd", kind="gated", m=777, n=3000, k=1400, act="gelu", bias=True,
             dtype="fp16"),
        # A prompt of 2048 tokens.
        dict(name="gated_prompt", kind="gated", m=2048, n=11008, k=4096, act="silu", bias=False,
             dtype="bf16"),
        # The norm in front of a block, one token. Latency.
        dict(name="norm_one", kind="norm", m=1, h=4096, norm="rms", residual=False, post=False,
             gate="none", alpha=1.0, out="int8", dtype="bf16", res="bf16"),
        # A step of 64 tokens: residual added, then the next block's norm.
        dict(name="norm_step", kind="norm", m=64, h=8192, norm="rms", residual=True, post=False,
             gate="none", alpha=1.0, out="int8", dtype="bf16", res="bf16"),
        # A block with norms on both sides, a gate for each channel and a scaled
        # residual, over a long prompt.
        dict(name="norm_prompt", kind="norm", m=8192, h=8192, norm="rms", residual=True, post=True,
             gate="channel", alpha=0.5, out="int8", dtype="bf16", res="bf16"),
        # LayerNorm with biases at an odd size, each token's own gate, a
        # residual kept in 32 bits, the result in 16 bits.
        dict(name="norm_layer", kind="norm", m=3001, h=1403, norm="layer", residual=True, post=True,
             gate="token", alpha=1.0, out="same", dtype="fp16", res="fp32"),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo: int, hi: int) -> int:
    """A layer's size: mostly a multiple of 128, else any."""
    v = _log_int(rng, lo, hi)
    return max(128, v // 128 * 128) if rng.random() < 0.7 else v


def draw(rng) -> dict:
    top = {c["name"]: work(c) for c in listed()}
    while True:
        kind = rng.choice(["linear", "linear", "gated", "norm"])
        dtype = rng.choice(["fp16", "bf16", "bf16"])
        if kind == "norm":
            residual = rng.random() < 0.7
            case = dict(kind=kind, m=_log_int(rng, 1, 16384), h=_size(rng, 64, 16384),
                        norm=rng.choice(["rms", "rms", "layer"]), residual=residual,
                        post=residual and rng.random() < 0.4,
                        gate=rng.choice(["none", "none", "channel", "token", "full"]) if residual
                        else "none", alpha=rng.choice([1.0, 0.5, 0.25]) if residual else 1.0,
                        out=rng.choice(["int8", "int8", "same"]), dtype=dtype, res=dtype)
            if residual and rng.random() < 0.25:
                case["res"] = "fp32"
            largest = top["norm_prompt"]
        else:
            case = dict(kind=kind, m=_log_int(rng, 1, 8192), n=_size(rng, 256, 28672),
                        k=_size(rng, 256, 16384), bias=rng.random() < 0.3,
                        dtype=rng.choice(["fp16", "bf16", "bf16", "fp32"]))
            if kind == "linear":
                case["xmode"] = rng.choice(["token", "token", "token", "tensor"])
                largest = top["linear_prompt"]
            else:
                case["act"] = rng.choice(["silu", "silu", "gelu", "gelu_tanh", "relu"])
                largest = top["gated_prompt"]
        cost = work(case)
        if cost["flops"] <= largest["flops"] and cost["bytes"] <= largest["bytes"]:
            return case


def work(case: dict) -> dict:
    m, e = case["m"], SIZE[case["dtype"]]
    if case["kind"] == "norm":
        h, r = case["h"], SIZE[case["res"]]
        b = m * h * e + 2 * e * h                               # x, weight, bias
        if case["residual"]:
            b += 2 * m * h * r + (2 * e * h if case["post"] else 0)
            b += e * {"none": 0, "channel": h, "token": m, "full": m * h}[case["gate"]]
        # codes and scales, and the values they stand for; or 16-bit values
        b += m * h * (1 + 1 + e) + 8 * m if case["out"] == "int8" else m * h * e
        return {"bytes": b, "flops": m * h * (8 + 6 * case["residual"] + 6 * case["post"])}
    n, k = case["n"], case["k"]
    two = 2 if case["kind"] == "gated" else 1
    return {"bytes": m * k + two * n * k + 4 * m + 4 * two * n * (1 + case["bias"]) + m * n * e,
            "flops": 2 * two * m * n * k}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _rows_to_codes(x):
    """INT8 codes of x's rows and their scales."""
    inv = 127 / x.abs().amax(1).clamp(min=EPS)
    return torch.round(x * inv[:, None]).clamp(-127, 127).to(torch.int8), 1 / inv


def _activations(rows: int, cols: int, g):
    """Hidden states: features of unequal size, a few tokens far larger than
    the others."""
    x = torch.randn(rows, cols, generator=g, device=DEV)
    x *= 0.5 + torch.rand(cols, generator=g, device=DEV)
    return x * (1 + 6 * (torch.rand(rows, 1, generator=g, device=DEV) < 0.03).float())


def prepare(case: dict, seed: int) -> dict:
    """What a serving program holds before the call: the layer's weights as
    codes and scales, and the activations that the step before left."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt, m = DTYPES[case["dtype"]], case["m"]
    st = dict(case=case)
    if case["kind"] == "norm":
        h = case["h"]
        st["x"] = _activations(m, h, g).to(dt)
        st["weight"] = (1 + 0.2 * torch.randn(h, generator=g, device=DEV)).to(dt)
        st["bias"] = (0.1 * torch.randn(h, generator=g, device=DEV)).to(dt)
        if case["residual"]:
            st["residual"] = (3 * _activations(m, h, g)).to(DTYPES[case["res"]])
            st["post_weight"] = (1 + 0.2 * torch.randn(h, generator=g, device=DEV)).to(dt)
            st["post_bias"] = (0.1 * torch.randn(h, generator=g, device=DEV)).to(dt)
            shape = {"none": None, "channel": (h,), "token": (m, 1), "full": (m, h)}[case["gate"]]
            st["gate"] = None
            if shape:
                st["gate"] = torch.sigmoid(torch.randn(shape, generator=g, device=DEV)).to(dt)
        if case["norm"] == "rms":
            st["bias"] = st["post_bias"] = None
        return st
    n, k = case["n"], case["k"]
    x = _activations(m, k, g)
    if case.get("xmode") == "tensor":
        codes, scale = _rows_to_codes(x.view(1, -1))
        st["x"], st["sx"] = codes.view(m, k), scale[0]
    else:
        st["x"], st["sx"] = _rows_to_codes(x)
    for name in ("w", "u") if case["kind"] == "gated" else ("w",):
        w = torch.empty(n, k, dtype=torch.int8, device=DEV)
        s = torch.empty(n, device=DEV)
        for r in range(0, n, 4096):
            part = slice(r, min(n, r + 4096))
            rows = torch.randn(part.stop - r, k, generator=g, device=DEV) / math.sqrt(k)
            w[part], s[part] = _rows_to_codes(rows)
        b = 0.1 * torch.randn(n, generator=g, device=DEV) if case["bias"] else None
        st.update({name: w, "s" + name: s, "b" + name: None if b is None else b.to(dt)})
    if own:
        from cublade_amd.quantization import QuantizedTensor
        zero = torch.zeros((), device=DEV)
        mode = "tensor" if st["sx"].dim() == 0 else "channel"
        st["qx"] = QuantizedTensor(st["x"], st["sx"], zero, mode, 0, 32, torch.int8, dt)
        for name in ("w", "u") if case["kind"] == "gated" else ("w",):
            st["q" + name] = QuantizedTensor(st[name], st["s" + name], zero, "channel", 0, 32,
                                             torch.int8, dt)
    return st


def run(st: dict):
    case = st["case"]
    if own:
        from cublade_amd.quantization import (dequantize_tensor, gated_w8a8, linear_w8a8,
                                              norm_tensor, residual_norm)
        if case["kind"] == "linear":
            return [linear_w8a8(st["qx"], st["qw"], st["bw"])]
        if case["kind"] == "gated":
            return [gated_w8a8(st["qx"], st["qw"], st["qu"], activation=case["act"],
                               gate_bias=st["bw"], up_bias=st["bu"])]
        to = torch.int8 if case["out"] == "int8" else st["x"].dtype
        if case["residual"]:
            h, q = residual_norm(st["x"], st["residual"], st["weight"], st["bias"],
                                 kind=case["norm"], eps=NORM_EPS, dtype=to,
                                 post_norm=case["post"],
                                 post_weight=st["post_weight"] if case["post"] else None,
                                 post_bias=st["post_bias"] if case["post"] else None,
                                 gate=st["gate"], scale=case["alpha"])
            return [h, dequantize_tensor(q) if case["out"] == "int8" else q]
        q = norm_tensor(st["x"], st["weight"], st["bias"], kind=case["norm"], eps=NORM_EPS,
                        dtype=to)
        return [dequantize_tensor(q) if case["out"] == "int8" else q]
    if case["kind"] == "norm":
        return _plain_norms(st)
    return [_plain_linear(st) if case["kind"] == "linear" else _plain_gated(st)]


# ---------------------------------------------------------------------------
# Plain forms: elementary torch operations in 32 bits
# ---------------------------------------------------------------------------
def _product(st: dict, w: str):
    x = st["x"].float() * st["sx"].reshape(-1, 1)
    y = x @ st[w].float().t() * st["s" + w]
    return y if st["b" + w] is None else y + st["b" + w].float()


def _plain_linear(st: dict):
    return _product(st, "w").to(DTYPES[st["case"]["dtype"]])


def _plain_gated(st: dict):
    g = _product(st, "w")
    act = st["case"]["act"]
    if act == "silu":
        a = g / (1 + torch.exp(-g))
    elif act == "gelu":
        a = 0.5 * g * (1 + torch.erf(g * math.sqrt(0.5)))
    elif act == "gelu_tanh":
        a = 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g)))
    else:
        a = g.clamp(min=0)
    return (a * _product(st, "u")).to(DTYPES[st["case"]["dtype"]])


def _plain_norm(x, norm: str, weight, bias):
    if norm == "layer":
        x = x - x.mean(1, keepdim=True)
    y = x * torch.rsqrt((x * x).mean(1, keepdim=True) + NORM_EPS) * weight.float()
    return y if bias is None else y + bias.float()


def _plain_norms(st: dict):
    case, x, out = st["case"], st["x"].float(), []
    if case["residual"]:
        if case["post"]:
            x = _plain_norm(x, case["norm"], st["post_weight"], st["post_bias"])
        if st["gate"] is not None:
            x = x * st["gate"].float()
        h = (st["residual"].float() + case["alpha"] * x).to(st["residual"].dtype)
        out, x = [h], h.float()
    y = _plain_norm(x, case["norm"], st["weight"], st["bias"])
    if case["out"] == "int8":
        inv = 127 / y.abs().amax(1, keepdim=True).clamp(min=EPS)
        y = torch.round(y * inv).clamp(-127, 127) * (1 / inv)
    return out + [y.to(DTYPES[case["dtype"]])]


# ---------------------------------------------------------------------------
# The results in 64 bits
# ---------------------------------------------------------------------------
def _exact_norm(rows, norm: str, weight, bias):
    """rows [m, h] in 64 bits; the moments by sums over the row."""
    h = rows.shape[1]
    mean = rows.sum(1) / h if norm == "layer" else torch.zeros_like(rows[:, 0])
    spread = (rows - mean[:, None]).square().sum(1) / h + NORM_EPS
    y = (rows - mean[:, None]) / spread.sqrt()[:, None] * weight.double()
    return y if bias is None else y + bias.double()


def exact(case: dict, seed: int):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    if case["kind"] == "norm":
        rows, out = st["x"].double(), []
        if case["residual"]:
            if case["post"]:
                rows = _exact_norm(rows, case["norm"], st["post_weight"], st["post_bias"])
            rows = rows * (1.0 if st["gate"] is None else st["gate"].double())
            h = st["residual"].double() + case["alpha"] * rows
            # the norm is that of the residual as it is stored
            out, rows = [h], h.to(st["residual"].dtype).double()
        y = _exact_norm(rows, case["norm"], st["weight"], st["bias"])
        if case["out"] == "int8":
            step = y.abs().amax(1).clamp(min=EPS)[:, None] / 127
            y = (y / step).round().clamp(-127, 127) * step
        return out + [y]
    m, n = case["m"], case["n"]
    y = torch.empty(m, n, dtype=torch.float64, device=DEV)
    x = st["x"].double()
    for c in range(0, n, 4096):                  # a block of output channels at a time
        cols = slice(c, min(n, c + 4096))

        def part(w):
            p = torch.matmul(x, st[w][cols].double().t().contiguous())   # whole numbers
            p = p * st["sx"].double().expand(m)[:, None] * st["s" + w][cols].double()
            return p if st["b" + w] is None else p + st["b" + w][cols].double()

        g = part("w")
        if case["kind"] == "gated":
            act = case["act"]
            if act == "silu":
                g = g * torch.sigmoid(g)
            elif act == "gelu":
                g = g * (1 - 0.5 * torch.erfc(g / math.sqrt(2)))
            elif act == "gelu_tanh":
                g = g * torch.sigmoid(math.sqrt(8 / math.pi) * (g + 0.044715 * g ** 3))
            else:
                g = torch.where(g > 0, g, torch.zeros_like(g))
            g = g * part("u")
        y[:, cols] = g
    return [y]
