"""Rows that are no whole chunks of 8 elements, of 4097 to 16384 elements: two elements of a
workgroup's thread per 8, many tokens and few (tests/_norms.py has the bounds)."""
from __future__ import annotations

import pytest
import torch

from tests import _norms as P
from tests import test_gpu_norms as T

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("hidden", [4097, 5001, 8189, 8193, 9001, 12345, 16383])
def test_norm(hidden, kind):
    from cublade_amd.quantization import norm_tensor
    i = hidden % 3
    dtype = (F32, F16, BF16)[i]
    for tokens in (3, 600):
        x = T._rand(tokens, hidden, seed=hidden, dtype=dtype, shift=0.3)
        w, b = (T._rand(hidden, seed=hidden + k, spread=0.3, shift=1.0, dtype=dtype) for k in (1, 2))
        zero = torch.zeros(x.shape, dtype=torch.float64)
        for bias in (None, b):
            y, err = P.norm(x.double(), zero, kind, 1e-5, w, bias)
            q = norm_tensor(*T._gpu(x, w, bias), kind=kind, eps=1e-5)
            P.check_codes(q.data, q.scale, y, err)
            n = norm_tensor(*T._gpu(x, w, bias), kind=kind, eps=1e-5, dtype=dtype)
            off = (n.cpu().double() - y).abs()
            assert bool((off <= (err + P.half(dtype) * y.abs()) * 1.01 + P.tiny(dtype)).all())


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("hidden", [5001, 8193, 12345, 16383])
def test_residual(hidden, post):
    T.test_residual(hidden, post)


def test_many_tokens_with_gates():
    """More than two tokens per CU, where these rows take two chunks from 4096 elements on."""
    from cublade_amd.quantization import residual_norm
    for hidden, tokens in ((4099, 530), (12345, 520)):
        x, r, g, w, pw = (T._rand(*s, seed=hidden + k, dtype=BF16) for k, s in
                          enumerate(((tokens, hidden), (tokens, hidden), (tokens, hidden), (hidden,), (hidden,))))
        for gate in (g, g[:, :1], g[0]):
            h, n = residual_norm(*T._gpu(x, r, w), post_norm=True, post_weight=pw.cuda(), gate=gate.cuda(), scale=0.5)
            want, bound = P.residual(x, r, "rms", 1e-6, True, pw, None, gate, 0.5, BF16)
            assert bool(((h.cpu().double() - want).abs() <= bound).all())
            P.check_codes(n.data, n.scale, *P.norm(h.cpu().double(), torch.zeros_like(want), "rms", 1e-6, w, None))


def test_rows_with_nan_and_infinity():
    from cublade_amd.quantization import norm_tensor
    for hidden in (4097, 9001, 16383):
        for tokens in (6, 600):
            x = T._rand(tokens, hidden, seed=6, dtype=F16)
            clean = norm_tensor(x.cuda())
            x[1, hidden // 2], x[3, 0], x[4, hidden - 1] = float("nan"), float("inf"), -float("inf")
            q = norm_tensor(x.cuda())
            bad = torch.zeros(tokens, dtype=torch.bool)
            bad[[1, 3, 4]] = True
            assert torch.equal(q.scale.cpu().isnan(), bad)
            assert torch.equal(q.data[~bad], clean.data[~bad]) and torch.equal(q.scale[~bad], clean.scale[~bad])
