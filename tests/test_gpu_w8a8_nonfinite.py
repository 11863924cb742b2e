"""A token that holds a NaN or an infinity leaves the W8A8 layers as NaN: its activations
are quantized with a NaN scale, in front of every product of a layer. The other tokens'
results are the bits of a call without it."""
from __future__ import annotations

import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
NAN, INF = float("nan"), float("inf")


def _x(tokens, features, dtype, seed=0):
    return torch.randn(tokens, features, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def _spoil(x):
    """A copy with a NaN, an infinity and a negative infinity in three tokens, and which."""
    bad = torch.zeros(x.shape[0], dtype=torch.bool, device=x.device)
    y, n = x.clone(), x.shape[1]
    for token, at, v in ((1, n // 2, NAN), (3, 0, INF), (4, n - 1, -INF), (6, n - 1, NAN)):
        y[token, at], bad[token] = v, True
    y[6, :] = NAN
    return y, bad


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows", [1, 7, 600])
def test_codes_of_tokens(rows, dtype):
    """The per-channel quantizer's bits, except that a token with a NaN or an infinity has a
    NaN scale and codes 0: every kernel that the row length chooses."""
    from cublade_amd.bindings.hip.quantize_int8 import quantize_per_channel_int8, quantize_tokens_int8
    for features in (1, 8, 30, 33, 56, 64, 100, 256, 1000, 1403, 2048, 2049, 2056, 4096, 5120, 8192,
                     11008, 16384, 20480, 65536, 70000) if rows < 100 else (8, 33, 100, 512, 1400, 4096):
        x = _x(rows, features, dtype, seed=features)
        want = quantize_per_channel_int8(x)
        assert all(torch.equal(a, b) for a, b in zip(quantize_tokens_int8(x), want)), features
        if rows == 1:
            continue
        y, bad = _spoil(x)
        q, s = quantize_tokens_int8(y)
        assert torch.equal(s.isnan(), bad) and not bool(q[bad].any()), features
        assert torch.equal(q[~bad], want[0][~bad]) and torch.equal(s[~bad], want[1][~bad]), features
    empty = quantize_tokens_int8(torch.zeros(rows, 0, dtype=dtype, device="cuda"))
    assert empty[0].shape == (rows, 0) and empty[1].shape == (rows,)


def _linear(n_in, n_out, dtype, bias):
    torch.manual_seed(n_in)
    return nn.Linear(n_in, n_out, bias=bias).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("features", [8, 64, 100, 1000, 1403, 2049, 4096, 5120, 8192, 11008, 20480, 70000])
def test_linear_layer(features, dtype):
    from cublade_amd.quantization import cuBladeW8A8LinearLayer
    layer = cuBladeW8A8LinearLayer.from_linear(_linear(features, 24, dtype, bias=features % 3 != 0))
    x = _x(8, features, dtype)
    clean = layer(x)
    y, bad = _spoil(x)
    got = layer(y)
    assert torch.equal(got.isnan(), bad[:, None].expand_as(got))
    assert torch.equal(got[~bad], clean[~bad])


def _mlp(hidden, inter, dtype, act):
    from cublade_amd.quantization import cuBladeW8A8GatedMLP
    return cuBladeW8A8GatedMLP(_linear(hidden, inter, dtype, True), _linear(hidden, inter, dtype, False),
                               _linear(inter, hidden, dtype, True), activation=act)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("hidden,inter", [(128, 344), (512, 1376), (100, 201)])
def test_gated_mlp(hidden, inter, act):
    from cublade_amd.quantization import norm_tensor
    mlp = _mlp(hidden, inter, BF16, act)
    x = _x(9, hidden, BF16)
    y, bad = _spoil(x)
    for clean, got in ((mlp(x), mlp(y)), (mlp(norm_tensor(x)), mlp(norm_tensor(y)))):
        assert torch.equal(got.isnan(), bad[:, None].expand_as(got))
        assert torch.equal(got[~bad], clean[~bad])


def test_block_keeps_the_token():
    """norm -> gated MLP -> residual -> the next norm's codes."""
    from cublade_amd.quantization import dequantize_tensor, norm_tensor, residual_norm
    mlp = _mlp(256, 640, F16, "silu")
    x, bad = _spoil(_x(8, 256, F16))
    h, q = residual_norm(mlp(norm_tensor(x)), torch.zeros_like(x))
    assert torch.equal(h.isnan(), bad[:, None].expand_as(h))
    assert torch.equal(dequantize_tensor(q).isnan(), bad[:, None].expand_as(h))


def test_outputs_past_fp16_do_not_come_back_finite():
    """A gated product past fp16's range is infinite: that token is NaN from the down
    projection on. Weights of 1/2, so g = u = 3.2 and 3200 for inputs of 0.1 and 100."""
    mlp = _mlp(64, 96, F16, "relu")
    for m in (mlp.gate, mlp.up, mlp.down):
        m.quantize(torch.full((m.out_features, m.in_features), 0.5, dtype=F16, device="cuda"))
    x = torch.full((4, 64), 0.1, dtype=F16, device="cuda")
    x[2] = 100
    assert mlp(x).isnan().all(1).tolist() == [False, False, True, False]
    assert bool(mlp(x)[[0, 1, 3]].isfinite().all())
