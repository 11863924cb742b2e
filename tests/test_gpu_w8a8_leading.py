"""A block on hidden states with leading dimensions, among them a decode step's [batch, 1,
hidden], whose codes are [tokens, hidden]: sums in the hidden states' shape, the values of
a call on flattened ones, and gates that repeat in every way."""
from __future__ import annotations

import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu

H = 256


def _rand(*shape, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).bfloat16().cuda()


@pytest.mark.parametrize("lead", [(5, 1), (3, 7), (2, 3, 4), (1, 1), (0, 4), ()])
def test_block(lead):
    from cublade_amd.quantization import (cuBladeW8A8GatedMLP, cuBladeW8A8LinearLayer, norm_tensor,
                                          residual_norm)
    torch.manual_seed(0)
    qkv = cuBladeW8A8LinearLayer.from_linear(nn.Linear(H, 3 * H).bfloat16().cuda())
    mlp = cuBladeW8A8GatedMLP(*(nn.Linear(a, b).bfloat16().cuda() for a, b in ((H, 640), (H, 640), (640, H))))
    w1, w2 = _rand(H, seed=1), _rand(H, seed=2)

    def block(x, attn_out):
        y = qkv(norm_tensor(x, w1))
        h, q = residual_norm(attn_out, x, w2)
        return y, h + mlp(q).view_as(h), h, q

    x, attn = _rand(*lead, H, seed=3), _rand(*lead, H, seed=4)
    y, out, h, q = block(x, attn)
    tokens = x.numel() // H
    assert y.shape == (tokens, 3 * H) and q.data.shape == (tokens, H) and h.shape == out.shape == x.shape
    flat = block(x.view(tokens, H), attn.view(tokens, H))
    assert torch.equal(flat[1].view_as(x), out) and torch.equal(flat[0], y)
    if len(lead) > 1 and tokens:       # a sum of the two shapes is refused here, where + would broadcast
        with pytest.raises(RuntimeError, match="residual"):
            residual_norm(mlp(q), h, w2)
    # tensors keep their leading dimensions
    assert qkv(x).shape == (*lead, 3 * H) and mlp(x).shape == x.shape


def test_gates_that_repeat():
    from cublade_amd.quantization import residual_norm
    x, r = _rand(3, 5, H, seed=5), _rand(3, 5, H, seed=6)
    for shape in ((3, 1, H), (1, 5, H), (3, 1, 1), (1, 5, 1), (3, 5, 1), (5, 1), (1, 1, H), (H,), (1,), ()):
        g = _rand(*shape, seed=7)
        full = g.expand(3, 5, H).contiguous()
        for a, b in zip(residual_norm(x, r, gate=g, dtype=torch.float32), residual_norm(x, r, gate=full, dtype=torch.float32)):
            assert torch.equal(a, b), shape


def test_layers_without_features():
    """No columns: the sums are empty and the bias is left."""
    from cublade_amd.quantization import cuBladeW8A8LinearLayer
    layer = cuBladeW8A8LinearLayer(0, 8, dtype=torch.float16).cuda()
    with torch.no_grad():
        layer.bias.copy_(torch.arange(8))
    y = layer(torch.zeros(2, 3, 0, dtype=torch.float16, device="cuda"))
    assert y.shape == (2, 3, 8) and torch.equal(y, layer.bias.detach().expand(2, 3, 8))
