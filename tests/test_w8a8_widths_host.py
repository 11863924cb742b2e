"""Inputs of W8A8 layers with a wrong number of features are refused before any work, also
empty ones and those whose elements would make whole rows."""
from __future__ import annotations

import pytest
import torch


@pytest.mark.parametrize("shape", [(48,), (2, 48), (4, 16), (2, 16), (2, 2, 8), (0, 48), (3, 0), (), (32, 1)])
def test_features_are_checked(shape):
    from cublade_amd.quantization import cuBladeW8A8GatedMLP, cuBladeW8A8LinearLayer
    layer = cuBladeW8A8LinearLayer(32, 8)
    mlp = cuBladeW8A8GatedMLP(layer, cuBladeW8A8LinearLayer(32, 8), cuBladeW8A8LinearLayer(8, 32))
    for m in (layer, mlp):
        with pytest.raises(ValueError, match="32 features"):
            m(torch.zeros(shape, dtype=torch.float16))
