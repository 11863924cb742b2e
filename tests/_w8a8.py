"""INT8 x INT8 products in 64 bits, and how far a kernel's result may be from them.

linear: the integer sum is exact, so the result is known to the last bit: the sum
rounded to fp32, times the token's scale, times the channel's, plus the bias, each
rounded to fp32, then rounded to the output's type.

gated: with u = 2^-24, g = act's argument has an error of at most
  e_g = 3 u |p| + u |p + b|         (p: the product without its bias)
(the sum's conversion, two scales, the bias), likewise e_u. |act'| <= 1.13 for all
four activations. The activation itself: v_exp_f32 and v_rcp_f32 are good to 1 ulp
(2 u); with z the sigmoid's argument, the rounding of z log2(e) (and of the constant)
costs |z| 2 u of e^-z, of which the sigmoid keeps at most |z| 2 u, plus 2 + 2 + 1 + 1
roundings. z itself is g (silu), or a polynomial of g with 4 roundings and two rounded
constants (6 u |z|, again no more than 6 u |z| of the sigmoid). So relative to act(g)
  r = (2 |z| + 6 |z| [tanh form] + 8) u.
gelu with erff (2 ulp at most, 4 u absolute since |erf| <= 1; its argument rounded
twice: at most 2 u |t| 2 / sqrt(pi) e^(-t^2) <= 1 u): (4 + 1 + 2) u / 2 |g| absolute,
taken as 4 u |g|. The product adds u. Last, one rounding to the output's type.
"""
from __future__ import annotations

import math

import torch

U = 2.0 ** -24
ACTS = ("silu", "gelu", "gelu_tanh", "relu")


def codes(rows: int, cols: int, seed: int, device="cuda", lo: int = -127):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(lo, 128, (rows, cols), generator=g, dtype=torch.int16).to(torch.int8)
    s = torch.rand(rows, generator=g) * 0.02 + 1e-3
    return q.to(device), s.to(device)


def sums(x, w):
    """Exact integer sums (|sum| < 2^53) as int64."""
    return (x.cpu().double() @ w.cpu().double().t()).long() if x.size(1) else \
        torch.zeros(x.size(0), w.size(0), dtype=torch.long)


def linear(x, sx, w, sw, bias, dtype):
    """The result to the last bit, on the CPU. Scales: [rows] or 0-d."""
    y = sums(x, w).float() * sx.cpu().expand(x.size(0))[:, None] * sw.cpu().expand(w.size(0))
    y = y + (0.0 if bias is None else bias.cpu().float())
    return y.to(dtype)


def _product(x, sx, w, sw, bias):
    p = sums(x, w).double() * sx.cpu().double().expand(x.size(0))[:, None] * \
        sw.cpu().double().expand(w.size(0))
    v = p if bias is None else p + bias.cpu().double()
    return v, 3 * U * p.abs() + U * v.abs()


def gated(x, sx, gate, up, act: str, dtype):
    """(result in 64 bits, bound of the kernel's error), on the CPU. gate, up:
    (codes, scales, bias or None)."""
    g, eg = _product(x, sx, *gate)
    u, eu = _product(x, sx, *up)
    if act == "silu":
        z, a = g, g * torch.sigmoid(g)
    elif act == "gelu_tanh":
        z = math.sqrt(8 / math.pi) * (g + 0.044715 * g ** 3)
        a = g * torch.sigmoid(z)
    elif act == "gelu":
        z, a = torch.zeros_like(g), 0.5 * g * torch.erfc(-g / math.sqrt(2))
    else:
        z, a = torch.zeros_like(g), g.clamp(min=0)
    own = a.abs() * (z.abs() * (8 if act == "gelu_tanh" else 2) + 8) * U
    if act == "gelu":
        own = 4 * U * g.abs()
    ea = 1.13 * eg + own
    y = a * u
    err = ea * u.abs() + a.abs() * eu + ea * eu + U * y.abs()
    # one rounding to the type, also of the erroneous value; fp16 below its normal range
    half = torch.finfo(dtype).eps / 2
    err = err * (1 + half) + half * y.abs() + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    return y, err + 1e-38


def qt(q, s, dtype=torch.float16):
    from cublade_amd.quantization import QuantizedTensor
    return QuantizedTensor(q, s, torch.zeros((), device=q.device),
                           "channel" if s.dim() else "tensor", 0, 32, torch.int8, dtype)
