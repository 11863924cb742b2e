"""INT8 activations times INT8 weights: linear_w8a8, gated_w8a8 and the layers
made of them (include/cublade_w8a8.h). No counterpart in the reference.

Both operands are QuantizedTensors as quantize_tensor makes them: activations
with a scale for each token (mode "channel", ch_axis 0 of [tokens, features]) or
one for all (mode "tensor"), weights with a scale for each output channel. The
integer sums are exact.
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn

from .quantizers import quantize_tensor
from .tensor import QuantizedTensor
from cublade_amd.bindings.hip.quantize_int8 import quantize_tokens_int8
from cublade_amd.bindings.hip.w8a8 import w8a8_gated, w8a8_linear


def _check(q: QuantizedTensor, name: str) -> None:
    if not isinstance(q, QuantizedTensor):
        raise ValueError(f"{name} must be a QuantizedTensor, got {type(q).__name__}")
    if q.dtype != torch.int8 or q.data.dtype != torch.int8:
        raise ValueError(f"{name} must hold torch.int8 codes, got {q.data.dtype}")
    if q.data.dim() != 2:
        raise ValueError(f"{name} must be 2-D, got {tuple(q.data.shape)}")
    if q.mode == "tensor":
        if q.scale.dim() != 0:
            raise ValueError(f"{name}: mode 'tensor' has one 0-d scale, got {tuple(q.scale.shape)}")
    elif q.mode != "channel" or q.axis not in (0, -2):
        raise ValueError(f"{name} must have one scale for each row (mode 'channel', axis 0) or one "
                         f"for all (mode 'tensor'), got mode '{q.mode}', axis {q.axis}")
    elif q.scale.dim() != 1:
        raise ValueError(f"{name}: mode 'channel' has [rows] scales, got {tuple(q.scale.shape)}")


def linear_w8a8(x: QuantizedTensor, weight: QuantizedTensor, bias: torch.Tensor | None = None,
                out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """x . weight^T + bias of quantized operands: y[m, n] = sx[m] sw[n]
    (sum_k qx[m, k] qw[n, k]) + bias[n].

    Args:
        x: INT8 [tokens, in_features], one scale for each token or one for all.
        weight: INT8 [out_features, in_features], one scale for each output
            channel or one for all.
        bias: [out_features], fp32, fp16 or bf16.
        out_dtype: fp32, fp16 or bf16; x.original_dtype by default.

    Returns [tokens, out_features]. The integer sums are exact (in_features at
    most 131071); scales and bias are applied in fp32, then one rounding to
    out_dtype. The result carries no gradient.

    Codes are read in place, but for rows that are not contiguous, more than 2^22
    bytes apart, or, with in_features a multiple of 16, at addresses that are none:
    those are copied in every call. in_features that is no multiple of 16 is slower;
    where it is no multiple of 4 either, both operands are copied in the call from
    640 tokens on.
    """
    _check(x, "x")
    _check(weight, "weight")
    return w8a8_linear(x.data, x.scale, weight.data, weight.scale, bias,
                       x.original_dtype if out_dtype is None else out_dtype)


def gated_w8a8(x: QuantizedTensor, gate: QuantizedTensor, up: QuantizedTensor, *,
               activation: str = "silu", gate_bias: torch.Tensor | None = None,
               up_bias: torch.Tensor | None = None,
               out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """act(x . gate^T + gate_bias) * (x . up^T + up_bias) in one kernel: the
    first half of a gated feed-forward block.

    Args:
        x, gate, up, out_dtype: as x, weight and out_dtype of linear_w8a8; gate
            and up have the same shape.
        activation: "silu", "gelu" (with the error function), "gelu_tanh" or
            "relu".
        gate_bias, up_bias: [out_features], of one dtype where both are given.

    Returns [tokens, out_features]. Neither projection is rounded before the
    product: fp32 from the integer sums on, one rounding to out_dtype. The
    result carries no gradient.
    """
    _check(x, "x")
    _check(gate, "gate")
    _check(up, "up")
    return w8a8_gated(x.data, x.scale, gate.data, gate.scale, up.data, up.scale, activation,
                      gate_bias, up_bias, x.original_dtype if out_dtype is None else out_dtype)


def _tokens(x, features: int):
    """(codes, scales, leading shape, dtype) of a layer's input: a tensor is
    quantized with one scale for each token, NaN where the token is not finite."""
    if isinstance(x, QuantizedTensor):
        _check(x, "x")
        if x.data.size(1) != features:
            raise ValueError(f"x must have {features} features, got {x.data.size(1)}")
        return x.data, x.scale, (x.data.size(0),), x.original_dtype
    if x.dim() == 0 or x.shape[-1] != features:
        raise ValueError(f"x must have {features} features, got {tuple(x.shape)}")
    rows = x.detach().reshape(math.prod(x.shape[:-1]), features)
    q, scale = quantize_tokens_int8(rows.contiguous())
    return q, scale, x.shape[:-1], x.dtype


class cuBladeW8A8LinearLayer(nn.Module):
    """nn.Linear with INT8 weights (one scale for each output channel) and INT8
    activations (one scale for each token, found in the call).

    The input is a fp16, bf16 or fp32 GPU tensor [..., in_features], whose leading
    dimensions the output keeps, or a QuantizedTensor [tokens, in_features] as
    norm_tensor gives it, which is taken as it is: its output is [tokens,
    out_features], to be viewed in the shape of the hidden states. The output has the input's (original) dtype. A token that holds
    a NaN or an infinity comes out as NaN.

    Storage: int8_weights int8 [out, in], scales float32 [out], bias parameter
    [out] in `dtype`, or None.
    """

    def __init__(self, in_features, out_features, bias=True, dtype=torch.bfloat16):
        super().__init__()
        self.in_features = in_features
        self.out_features = out_features
        self.register_buffer("int8_weights",
                             torch.empty(out_features, in_features, dtype=torch.int8))
        self.register_buffer("scales", torch.ones(out_features, dtype=torch.float32))
        self.bias = nn.Parameter(torch.zeros(out_features, dtype=dtype)) if bias else None

    def _apply(self, fn, recurse=True):
        # the scales stay float32 where a model is cast (module.half())
        scales = self.scales
        super()._apply(fn, recurse)
        if self.scales.dtype != torch.float32:
            self.scales = scales.to(self.scales.device)
        return self

    @torch.no_grad()
    def quantize(self, weight_fp: torch.Tensor):
        """Quantize a [out, in] weight per output channel (INT8, symmetric), on
        the GPU; the codes go to the weight's device."""
        if tuple(weight_fp.shape) != (self.out_features, self.in_features):
            raise ValueError(f"weight must be [{self.out_features}, {self.in_features}], got "
                             f"{tuple(weight_fp.shape)}")
        w = weight_fp.detach()
        qt = quantize_tensor((w if w.is_cuda else w.cuda()).contiguous(), dtype=torch.int8,
                             mode="channel", ch_axis=0)
        self.int8_weights = qt.data.to(w.device)
        self.scales = qt.scale.to(w.device)

    @classmethod
    def from_linear(cls, linear: nn.Linear) -> "cuBladeW8A8LinearLayer":
        layer = cls(linear.in_features, linear.out_features, bias=linear.bias is not None,
                    dtype=linear.weight.dtype)
        layer.quantize(linear.weight)
        if linear.bias is not None:
            layer.bias = linear.bias
        return layer

    def forward(self, x):
        q, scale, lead, dtype = _tokens(x, self.in_features)
        y = w8a8_linear(q, scale, self.int8_weights, self.scales, self.bias, dtype)
        return y.view(*lead, self.out_features)


class cuBladeW8A8GatedMLP(nn.Module):
    """down(act(gate(x)) * up(x)) with W8A8 layers: the tokens are quantized
    once for both projections, which run as one kernel (gated_w8a8).

    gate, up, down: nn.Linear (quantized here) or cuBladeW8A8LinearLayer. The
    input is that of cuBladeW8A8LinearLayer.
    """

    def __init__(self, gate, up, down, activation: str = "silu"):
        super().__init__()
        if (gate.in_features, gate.out_features) != (up.in_features, up.out_features) or \
                down.in_features != up.out_features:
            raise ValueError("gate and up must have one shape, and down their outputs as inputs")
        self.gate, self.up, self.down = (
            cuBladeW8A8LinearLayer.from_linear(m) if isinstance(m, nn.Linear) else m
            for m in (gate, up, down))
        self.activation = activation

    def forward(self, x):
        q, scale, lead, dtype = _tokens(x, self.gate.in_features)
        h = w8a8_gated(q, scale, self.gate.int8_weights, self.gate.scales, self.up.int8_weights,
                       self.up.scales, self.activation, self.gate.bias, self.up.bias, dtype)
        return self.down(h).view(*lead, self.down.out_features)
