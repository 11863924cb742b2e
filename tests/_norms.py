"""norm_tensor and residual_norm in 64 bits, with bounds of the kernel's error.

u = 2^-24 (half a step of fp32). Sums of n terms in any order: an error of at most
(n - 1) u of the sum of magnitudes; here n counts the longest chain of the kernel, at
most c = hidden, which is taken.

A norm of v (error e of each element on entry, zero for tensors that are read):
  layer: mean m: |dm| <= mean e + (c + 1) u mean|v|; d = v - m: e + |dm| + u |d|
  ss = sum d^2: relative error 2 max over the row of (error of d, as a norm) ...
To stay simple the bound is a norm-wise one: with D the 2-norm of d and E the 2-norm
of its errors, rstd = (D^2 / n + eps)^(-1/2) is off by a factor of at most
  1 + E / D + (c / 2 + 4) u     (sum, division, eps, v_rsq_f32's 1 ulp)
unless D is tiny beside eps, where the factor is closer to 1 still. Then
  |dn| <= |n| (E / D + (c / 2 + 8) u) + |w| rstd e_d + 2 u |n + b|.
E / D <= 1 is asserted (rows whose values all but vanish beside their mean are not
among the cases).
h = r + alpha gate t: |dh| <= alpha gate (dt + 3 u |t|) + u |h|, then one rounding to
h's type; n is the norm of h as stored, so the kernel's own h is taken from there on
and dh does not go on. The result: 16 bits, one more rounding; codes: the scale is off
by d(amax) / 127 + 3 u scale, and the value code * scale by half a step more: a value
next to the middle of two codes may take either.
"""
from __future__ import annotations

import torch

U = 2.0 ** -24


def half(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def tiny(dtype) -> float:
    return 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134


def norm(v, e, kind, eps, w, b):
    """(norm in 64 bits, bound of its error) of rows v with errors up to e."""
    n = v.shape[1]
    d, ed = v, e
    if kind == "layer":
        m = v.sum(1, keepdim=True) / n
        dm = e.sum(1, keepdim=True) / n + (n + 1) * U * v.abs().sum(1, keepdim=True) / n
        d = v - m
        ed = e + dm + U * (d.abs() + dm)
    D2 = d.square().sum(1, keepdim=True)
    rstd = (D2 / n + eps).rsqrt()
    E = ed.square().sum(1, keepdim=True).sqrt()
    share = E / D2.clamp(min=1e-300).sqrt() * (D2 > 0)
    assert bool((share[D2 > 0] <= 1).all())
    w = torch.ones(n, dtype=torch.float64) if w is None else w.double()
    y = d * rstd * w
    err = y.abs() * (share + (n / 2 + 8) * U) * 1.01 + w.abs() * rstd * ed * 1.01
    y = y if b is None else y + b.double()
    return y, err + 2 * U * y.abs()


def residual(x, r, kind, eps, post, pw, pb, gate, alpha, dtype):
    """(h in 64 bits, bound, among them the rounding to dtype)."""
    t, e = x.double(), torch.zeros(x.shape, dtype=torch.float64)
    if post:
        t, e = norm(t, e, kind, eps, pw, pb)
    if gate is not None:
        t, e = t * gate.double(), (e + U * t.abs()) * gate.double().abs()
    h = r.double() + alpha * t
    e = abs(alpha) * (e + 2 * U * t.abs()) + U * h.abs()
    return h, (e + half(dtype) * h.abs()) * 1.01 + tiny(dtype)


def check_codes(got, scale, y, err):
    """Codes and scales of y (64 bits, errors up to err) within their bounds."""
    got, scale = got.cpu(), scale.cpu().double()
    amax, e = y.abs().amax(1), err.amax(1)
    want = amax.clamp(min=1e-12) / 127
    assert bool(((scale - want).abs() <= e / 127 + 4 * U * want).all())
    assert int(got.abs().max()) <= 127
    off = (got.double() * scale[:, None] - y).abs()
    bound = scale[:, None] * (0.5 + 127 * 4 * U) + err + (e / 127)[:, None]
    assert bool((off <= bound).all()), float((off / bound).max())
    # every token uses the whole range
    full = amax > 1e-9
    assert bool((got.abs().amax(1)[full] == 127).all())
