"""examples/quantized_decode.py: a layer with W8A16 projections and the 8-bit
cache follows the unquantised fp32 layer.

Bound on the relative error of the outputs (root mean square): INT8 weights with
one scale per row of Gaussian-like values err by half a step of 1 / 127 of about
3.5 standard deviations, uniformly: 3.5 / 127 / sqrt(12) = 0.8% of a value's
standard deviation, in the projections of q, k, v and of the output; the cache's
INT8 codes by as much (up to twice where a page's scale has grown), its FP8 codes
by 2^-4 / sqrt(3) = 3.6% at most; bf16 roundings by 0.2% each. q's, k's and v's
errors and the output projection's add up to at most 0.8% * 4 + 1.6% * 2 + 1% =
7.4% for INT8 and 0.8% * 4 + 3.6% * 2 + 1% = 11.4% for FP8 (logits are of order
1, so an error of a score is one of its weight's relative error)."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("store,bound", [(torch.int8, 0.074), (torch.float8_e4m3fn, 0.114)])
def test_layer_follows_fp32(store, bound):
    path = Path(__file__).resolve().parents[1] / "examples" / "quantized_decode.py"
    spec = importlib.util.spec_from_file_location("quantized_decode", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    err = mod.run(store)
    assert 0 < err <= bound, err
