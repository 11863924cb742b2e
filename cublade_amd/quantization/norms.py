"""The norms before and after a block: norm_tensor and residual_norm, one kernel
each (include/cublade_w8a8.h). No counterpart in the reference.

Their results are the activations of the INT8 products (linear_w8a8, gated_w8a8
and the layers made of them): INT8 codes with one scale for each token, found
while the token is at hand, so that it is not written in 16 bits and read again.
"""
from __future__ import annotations

import torch

from .quantizers import _zero_scalar
from .tensor import QuantizedTensor
from cublade_amd.bindings.hip.norm import norm


def _result(x: torch.Tensor, out, scale):
    if out is None:
        return None
    if scale is None:
        return out.view(x.shape)
    return QuantizedTensor(out, scale, _zero_scalar(x.device), "channel", 0, 32, torch.int8, x.dtype)


def norm_tensor(x: torch.Tensor, weight: torch.Tensor | None = None,
                bias: torch.Tensor | None = None, *, kind: str = "rms", eps: float = 1e-6,
                dtype: torch.dtype = torch.int8):
    """norm(x) over the last dimension, quantized: the norm in front of a block.

    Args:
        x: [..., hidden], fp32, fp16 or bf16; rows are read in place.
        weight, bias: [hidden], of one dtype (fp32, fp16 or bf16); None: 1 and 0.
        kind: "rms", x / sqrt(mean(x^2) + eps), or "layer", (x - mean) /
            sqrt(var + eps).
        dtype: torch.int8, or a floating-point type for the result as it is.

    Returns a QuantizedTensor [tokens, hidden] with one scale for each token
    (leading dimensions are flattened), as quantize_tensor(mode="channel") makes
    it of the norm in fp32, and original_dtype x's; or a tensor like x in `dtype`.
    Sums and the norm are fp32 (the sum of squares of elements beyond about 2^63
    overflows, and the result is 0); their order, and so a result's last bits, may
    differ with the number of tokens and the tensors' alignment. A token with a NaN or
    an infinity, in x or in the norm, gets a NaN scale and reads back as NaN. The
    result carries no gradient.
    """
    if dtype is None:
        raise ValueError("norm_tensor: dtype is None")
    _, out, scale = norm(x, None, weight, bias, kind, eps, dtype, False, None, None, None, 1.0)
    return _result(x, out, scale)


def residual_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor | None = None,
                  bias: torch.Tensor | None = None, *, kind: str = "rms", eps: float = 1e-6,
                  dtype: torch.dtype | None = torch.int8, post_norm: bool = False,
                  post_weight: torch.Tensor | None = None, post_bias: torch.Tensor | None = None,
                  gate: torch.Tensor | None = None, scale: float = 1.0):
    """What lies between a block's output x and the next block's input: with t =
    norm(x) post_weight + post_bias if post_norm, else x,

        h = residual + scale * gate * t,        n = norm(h) weight + bias

    Args:
        x: as in norm_tensor; residual: x's shape, x's dtype or fp32.
        weight, bias, kind, eps: of the next block's norm (kind and eps of both);
            dtype: of n, as in norm_tensor, or None: h only.
        post_norm, post_weight, post_bias: the norm after the block. All weights
            and biases have one dtype.
        gate: any shape that broadcasts to x's (of a channel, of a token, of
            both), fp32, fp16 or bf16. One that repeats some tokens' rows but not
            all (as [batch, 1, hidden] does) is expanded to x's size in the call.
        scale: of the block's part of the sum.

    Returns (h, n): h in x's shape and the residual's dtype, n as norm_tensor
    (h) gives it: n is taken of h as rounded to its dtype; as codes it is [tokens,
    hidden], its leading dimensions flattened. Neither carries a gradient.
    """
    h, out, s = norm(x, residual, weight, bias, kind, eps, dtype, post_norm, post_weight, post_bias,
                     gate, float(scale))
    return h, _result(x, out, s)
