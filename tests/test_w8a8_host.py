"""Refusals of the INT8 x INT8 products and of the norms around a block (no GPU work): C
entries, bindings, layers."""
from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest
import torch
import torch.nn as nn

from tests import _w8a8 as P

ROOT = Path(__file__).resolve().parents[1]


def _L():
    from cublade_amd import _abi
    return _abi, _abi.lib()


def test_header_and_signatures_agree():
    _abi, L = _L()
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "cublade_w8a8.h").read_text(), flags=re.S)
    names = set(re.findall(r"\b(cbq_\w+)\s*\(", text))
    assert names == set(_abi.W8A8_SIGNATURES) and all(hasattr(L, n) for n in names)


def _refused(rc, needle):
    _, L = _L()
    assert rc == 1 and needle in L.cbq_last_error().decode(), L.cbq_last_error()


def test_c_entries_refuse_bad_arguments():
    _abi, L = _L()
    by = ctypes.byref

    def rows(data=4096, stride=64, scale=4096, step=1):
        return by(_abi.I8Rows(data, stride, scale, step))

    def linear(x=None, w=None, bias=None, bdt=0, m=200, n=8, k=64, y=4096, out=1, ws=None, nb=0):
        return L.cbq_w8a8_linear(x or rows(), w or rows(), bias, bdt, m, n, k, y, out, ws, nb, None)

    def gated(gate=None, up=None, act=0, **kw):
        a = dict(m=200, n=8, k=64, out=1)
        a.update(kw)
        return L.cbq_w8a8_gated(rows(), gate or rows(), up or rows(), None, None, 0, act, a["m"],
                                a["n"], a["k"], 4096, a["out"], None, 0, None)

    _refused(linear(m=-1), "negative")
    _refused(linear(m=1 << 31), "2^31")
    _refused(linear(k=131072, x=rows(stride=131072), w=rows(stride=131072)), "131071")
    _refused(linear(out=3), "out_dtype")
    _refused(linear(bias=4096, bdt=3), "bias dtype")
    _refused(linear(x=rows(data=None)), "x has a null")
    _refused(linear(w=rows(scale=None)), "w has a null")
    _refused(linear(x=rows(stride=63)), "bytes apart")
    _refused(linear(w=rows(stride=(1 << 22) + 16)), "bytes apart")
    _refused(linear(x=rows(step=2)), "scale_stride")
    _refused(linear(y=None), "y is null")
    _refused(linear(y=4097), "aligned")
    _refused(linear(m=1 << 20, n=1 << 13, k=8), "2^32")
    _refused(gated(act=4), "activation")
    _refused(gated(act=-1), "activation")
    _refused(gated(up=rows(scale=None)), "up has a null")
    _refused(gated(gate=rows(stride=8)), "gate rows")
    # nothing to compute: no pointer is looked at
    none = by(_abi.I8Rows(None, 0, None, 0))
    assert L.cbq_w8a8_linear(none, rows(), None, 0, 0, 8, 64, None, 1, None, 0, None) == 0
    assert L.cbq_w8a8_linear(rows(), none, None, 0, 8, 0, 64, None, 1, None, 0, None) == 0


def test_norm_entry_refuses_bad_arguments():
    _abi, L = _L()

    def norm(**kw):
        a = dict(tokens=4, hidden=64, x=4096, x_stride=64, out=4096, scale=4096, x_dtype=1,
                 residual_dtype=1, out_dtype=_abi.I8)
        a.update(kw)
        return L.cbq_norm(ctypes.byref(_abi.NormArgs(**a)), None)

    res = dict(residual=4096, residual_stride=64, h=4096)
    assert L.cbq_norm(None, None) == 1
    _refused(norm(tokens=-1), "negative")
    _refused(norm(hidden=1 << 31), "2^31")
    _refused(norm(x_dtype=3), "x dtype")
    _refused(norm(residual_dtype=2, **res), "residual must")
    _refused(norm(out_dtype=4), "out dtype")
    _refused(norm(weight=4096, param_dtype=3), "parameter dtype")
    _refused(norm(gate=4096, gate_dtype=7, **res), "gate dtype")
    _refused(norm(kind=2), "kind")
    _refused(norm(post=1), "need a residual")
    _refused(norm(gate=4096), "need a residual")
    _refused(norm(post_weight=4096, **res), "need post")
    _refused(norm(gate=4096, gate_channel_stride=2, **res), "gate_channel_stride")
    _refused(norm(gate=4096, gate_token_stride=-1, **res), "gate_token_stride")
    _refused(norm(x=None), "null")
    _refused(norm(out=None), "null")
    _refused(norm(residual=4096, residual_stride=64), "null")
    _refused(norm(scale=None), "scale")
    _refused(norm(x_stride=63), "closer")
    _refused(norm(residual=4096, residual_stride=8, h=4096), "closer")
    for name in ("x", "weight", "bias", "residual", "h"):
        _refused(norm(**{**res, name: 4097}, param_dtype=1), "aligned")
    _refused(norm(out=4098, out_dtype=0), "aligned")
    assert norm(tokens=0, x=None) == 0 and norm(hidden=0, x=None) == 0


def test_norm_arguments_as_bytes():
    """The binding packs cbq_norm_args itself: the same bytes as the structure's."""
    from cublade_amd import _abi
    from cublade_amd.bindings.hip.norm import _ARGS
    assert _ARGS.size == ctypes.sizeof(_abi.NormArgs)
    values = [*range(1, 24), 0.5, -2.0]
    assert _ARGS.pack(*values) == bytes(_abi.NormArgs(*values))


def test_norms_on_the_host():
    from cublade_amd.quantization import norm_tensor, residual_norm
    x = torch.zeros(4, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        norm_tensor(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        residual_norm(x, x)
    with pytest.raises(ValueError, match="None"):
        norm_tensor(x, dtype=None)


def test_workspace_sizes():
    _abi, L = _L()
    C = _abi.WS_CTRL_BYTES
    assert L.cbq_w8a8_ws_bytes(64, 11008, 4096, 1) == C           # few rows: none
    assert L.cbq_w8a8_ws_bytes(128, 4096, 4096, 2) == C
    assert L.cbq_w8a8_ws_bytes(4096, 28672, 8192, 1) == C        # tiles enough for every CU
    assert L.cbq_w8a8_ws_bytes(0, 8, 8, 1) == C and L.cbq_w8a8_ws_bytes(1000, 8, 0, 2) == C
    # many tokens with rows of 1403 codes: copies in rows of 1408
    for p in (1, 2):
        assert L.cbq_w8a8_ws_bytes(4096, 8192, 1403, p) == C + 1408 * (4096 + p * 8192)
    # few tiles of long rows: planes of int32 sums (here of whole tiles), for each projection
    one, two = (L.cbq_w8a8_ws_bytes(2304, 256, 11008, p) - C for p in (1, 2))
    assert one % (2304 * 256 * 4) == 0 and two % (2 * 2304 * 256 * 4) == 0
    assert 2 <= one // (2304 * 256 * 4) <= 8 and 2 <= two // (2 * 2304 * 256 * 4) <= 8
    # a small product by another kernel, which cuts nothing
    assert L.cbq_w8a8_ws_bytes(256, 1024, 11008, 1) == C


def test_quantized_operands_are_checked():
    from cublade_amd.quantization import QuantizedTensor, gated_w8a8, linear_w8a8
    (x, sx), (w, sw) = P.codes(4, 32, 1, "cpu"), P.codes(8, 32, 2, "cpu")
    qx, qw = P.qt(x, sx), P.qt(w, sw)
    zero = torch.zeros(())

    def q(data=x, scale=sx, mode="channel", axis=0, dtype=torch.int8):
        return QuantizedTensor(data, scale, zero, mode, axis, 32, dtype, torch.float16)

    for bad, needle in ((x, "QuantizedTensor"), (q(dtype=torch.float8_e4m3fn), "int8"),
                        (q(data=x.float()), "int8"), (q(mode="group"), "row"), (q(axis=1), "row"),
                        (q(data=x.view(2, 2, 32)), "2-D"), (q(scale=sx[0]), "scales"),
                        (q(mode="tensor"), "0-d")):
        with pytest.raises(ValueError, match=needle):
            linear_w8a8(bad, qw)
        with pytest.raises(ValueError, match=needle):
            linear_w8a8(qx, bad)
        with pytest.raises(ValueError, match=needle):
            gated_w8a8(qx, qw, bad)
    with pytest.raises(RuntimeError, match="CUDA"):
        linear_w8a8(qx, qw)
    with pytest.raises(RuntimeError, match="CUDA"):
        gated_w8a8(qx, qw, qw)


def test_layers_on_the_host():
    from cublade_amd.quantization import cuBladeW8A8GatedMLP, cuBladeW8A8LinearLayer
    layer = cuBladeW8A8LinearLayer(32, 8, dtype=torch.float16)
    assert layer.half().scales.dtype == torch.float32 and layer.bias.dtype == torch.float16
    assert set(layer.state_dict()) == {"int8_weights", "scales", "bias"}
    with pytest.raises(ValueError, match=r"\[8, 32\]"):
        layer.quantize(torch.zeros(32, 8))
    with pytest.raises(RuntimeError, match="CUDA"):
        layer(torch.zeros(2, 32))
    (x, sx) = P.codes(4, 16, 1, "cpu")
    with pytest.raises(ValueError, match="32 features"):
        layer(P.qt(x, sx))
    with pytest.raises(ValueError, match="one shape"):
        cuBladeW8A8GatedMLP(layer, cuBladeW8A8LinearLayer(32, 9), cuBladeW8A8LinearLayer(9, 32))
    with pytest.raises(ValueError, match="one shape"):
        cuBladeW8A8GatedMLP(layer, cuBladeW8A8LinearLayer(32, 8), nn.Linear(9, 32))
