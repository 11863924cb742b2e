"""Refusals of the token quantizer of the W8A8 layers (no GPU work)."""
from __future__ import annotations

import pytest
import torch


def test_c_entry_refuses_bad_arguments():
    from cublade_amd import _abi
    L = _abi.lib()

    def call(x=4096, dtype=1, rows=4, cols=8, q=4096, scale=4096):
        return L.cbq_quant_int8_tokens(x, dtype, rows, cols, 1e-12, None, 0, q, scale, None)

    for kw, needle in ((dict(dtype=3), "dtype"), (dict(rows=-1), "negative"), (dict(cols=-1), "negative"),
                       (dict(x=None), "null"), (dict(q=None), "null"), (dict(scale=None), "null"),
                       (dict(rows=1 << 31), "too many rows")):
        assert call(**kw) == 1 and needle in L.cbq_last_error().decode()
    assert call(rows=0, x=None) == 0 and call(cols=0, q=None) == 0


def test_binding_refuses_bad_tensors():
    from cublade_amd.bindings.hip.quantize_int8 import quantize_tokens_int8
    with pytest.raises(RuntimeError, match="CUDA"):
        quantize_tokens_int8(torch.zeros(2, 8))
