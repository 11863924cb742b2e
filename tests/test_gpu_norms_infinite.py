"""A norm that is infinite or NaN without the token being so (an infinite weight or bias, a
product past fp32): a NaN scale and codes 0, as where the token itself is not finite."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hidden", [64, 1000, 1403, 4096, 8200, 9001, 20000, 40000])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_scale_is_nan(hidden, kind):
    from cublade_amd.quantization import dequantize_tensor, norm_tensor, residual_norm
    g = torch.Generator().manual_seed(hidden)
    x = torch.randn(3, hidden, generator=g).half().cuda()
    ones, inf = torch.ones(hidden, device="cuda"), float("inf")
    large = ones * 3.4e38
    x[:, 7] = 30.0                                  # its norm passes 1 for sure
    at = ones.clone()
    at[hidden - 1] = inf
    for kw in (dict(weight=at), dict(bias=at), dict(bias=-at), dict(weight=ones, bias=at), dict(weight=large)):
        for q in (norm_tensor(x, kind=kind, **kw), residual_norm(x, torch.zeros_like(x), kind=kind, **kw)[1]):
            assert bool(q.scale.isnan().all()) and not bool(q.data.any()), kw.keys()
            assert bool(dequantize_tensor(q).isnan().all())
    q = norm_tensor(x, ones, kind=kind)
    assert bool(q.scale.isfinite().all())
