"""GELU with the error function where its gate is far below zero: the activation keeps its
digits (1 + erf cancels there: at -5 within 5%, below -5.6 it is 0).

With u = 2^-24, g = p + b (p: the product, b: the bias) has an error of at most e_g = 3 u |p|
+ u |g|. a = g / 2 erfc(t), t = -g / sqrt(2). For g < 0: |a'| <= |a| (1 / |g| + phi(g) / Phi(g)),
and phi / Phi <= (|g| + sqrt(g^2 + 4)) / 2 <= |g| + 1 / |g|, so e_g costs at most |a| e_g (|g| +
2 / |g|); second orders are below 1% of that here. t has two roundings (the constant and the
product), 2 u |t|, and |t erfc'(t) / erfc(t)| <= t (t + sqrt(t^2 + 2)) <= 2 t^2 + 1 = g^2 + 1.
erfcf is good to 16 ulp (OpenCL's limit for it), 32 u; the product one rounding more. Together
  e_a = |a| (1.01 e_g (|g| + 2 / |g|) + u (2 (g^2 + 1) + 33)).
The up projection and the product as in tests/_w8a8.py."""
from __future__ import annotations

import math

import pytest
import torch

from tests import _w8a8 as P
from tests import _w8a8_forms as F

pytestmark = pytest.mark.gpu


# few rows, one output per thread, tiles, K in ranges
@pytest.mark.parametrize("m,n,k", [(1, 300, 256), (40, 129, 1001), (3, 70, 9), (2100, 260, 272), (700, 300, 1001),
                                   (2304, 256, 11008)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tail(m, n, k, dtype):
    from cublade_amd.quantization import gated_w8a8
    if m == 2304:
        f = F.form(m, n, k, 2)
        assert f.kernel == F.TILES and f.ranges > 1
    (x, sx), (g, sg), (w, sw) = (P.codes(r, k, s) for r, s in ((m, 1), (n, 2), (n, 3)))
    # gates of -5.5 with products within 2.5 of it; up projections of some thousands
    p = P.sums(x, g).double()
    sx, sg = torch.full((m,), 1.0, device="cuda"), torch.full((n,), 2.5 / float(p.abs().max()), device="cuda")
    bias = torch.full((n,), -5.5, device="cuda")
    y = gated_w8a8(P.qt(x, sx, dtype), P.qt(g, sg), P.qt(w, sw), activation="gelu", gate_bias=bias).cpu().double()
    p = p * sg[0].double().cpu()
    v = p - 5.5
    assert float(v.max()) < -2.9 and float(v.min()) > -8.1
    up = P.sums(x, w).double() * sw.cpu().double()
    a = 0.5 * v * torch.erfc(-v / math.sqrt(2))
    eg = 3 * P.U * p.abs() + P.U * v.abs()
    ea = a.abs() * (1.01 * eg * (v.abs() + 2 / v.abs()) + P.U * (2 * (v.square() + 1) + 33))
    eu = 4 * P.U * up.abs()
    want = a * up
    half = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    err = (ea * up.abs() + a.abs() * eu + ea * eu + P.U * want.abs()) * (1 + half) + half * want.abs()
    off = (y - want).abs()
    assert bool((off <= err).all()), float((off / err.clamp(min=1e-300)).max())
