"""The norms before and after a block on the HIP C ABI (include/cublade_w8a8.h).
No counterpart in the reference."""
from __future__ import annotations

import math
import struct

import torch

from ... import _abi


# cbq_norm_args as bytes (a ctypes.Structure of 25 fields takes 1 us more to make).
_ARGS = struct.Struct("<qqQqQqQqqQQQQQQQiiiiiiiff4x")


def _rows(x: torch.Tensor, hidden: int) -> tuple[torch.Tensor, int]:
    """x (not empty) as [tokens, hidden] whose rows the kernel can read in place,
    and the elements from one row to the next."""
    if x.dim() != 2:
        x = x.reshape(-1, hidden)
    tokens, stride = x.size(0), x.stride()
    if tokens > 1 and stride[0] < hidden or hidden > 1 and stride[1] != 1:
        return x.contiguous(), hidden
    return x, stride[0] if tokens > 1 else hidden


def _param(p: torch.Tensor | None, hidden: int, dev: torch.device, dtype, name: str):
    """(data pointer or 0, the tensor it points to, the parameters' dtype)."""
    if p is None:
        return 0, None, dtype
    if p.device != dev or p.dtype not in _abi.DTYPE_CODE or p.dim() != 1 or p.numel() != hidden:
        raise RuntimeError(f"{name} must be [{hidden}] in float32, float16 or bfloat16 on {dev}, "
                           f"got {tuple(p.shape)} {p.dtype} on {p.device}")
    if dtype is not None and p.dtype != dtype:
        raise RuntimeError(f"the weights and biases must have one dtype, got {dtype} and {p.dtype} "
                           f"for {name}")
    if p.stride(0) != 1:
        p = p.contiguous()
    return p.data_ptr(), p, p.dtype


def norm(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor | None,
         bias: torch.Tensor | None, kind: str, eps: float, dtype: torch.dtype | None, post: bool,
         post_weight: torch.Tensor | None, post_bias: torch.Tensor | None,
         gate: torch.Tensor | None, alpha: float):
    """(h or None, codes or values [tokens, hidden] or None, scales or None); see
    quantization.norms."""
    if not x.is_cuda:
        raise RuntimeError(f"x must be on CUDA, got {x.device}")
    codes = _abi.DTYPE_CODE
    x_dtype = x.dtype
    code = codes.get(x_dtype)
    if code is None:
        raise RuntimeError(f"x must be float32, float16 or bfloat16, got {x_dtype}")
    shape = x.shape
    if not shape:
        raise RuntimeError("x must have at least 1 dimension")
    k = _abi.NORM_CODE.get(kind)
    if k is None:
        raise RuntimeError(f"kind must be one of {sorted(_abi.NORM_CODE)}, got {kind!r}")
    dev, hidden = x.device, shape[-1]
    out_code = _abi.I8 if dtype is torch.int8 else codes.get(dtype)
    if out_code is None:
        if dtype is not None:
            raise RuntimeError(f"dtype must be int8, float32, float16 or bfloat16, got {dtype}")
        out_code = 0
    tokens = shape[0] if len(shape) == 2 else math.prod(shape[:-1])
    h, r_code = None, code
    if residual is not None:
        r_dtype = residual.dtype
        if residual.shape != shape or residual.device != dev or (
                r_dtype != x_dtype and r_dtype != torch.float32):
            raise RuntimeError(f"residual must be {tuple(shape)} in x's dtype or float32 on {dev}, "
                               f"got {tuple(residual.shape)} {r_dtype} on {residual.device}")
        r_code = codes[r_dtype]
        h = x.new_empty(shape, dtype=r_dtype)
    elif post or gate is not None:
        raise RuntimeError("a gate and a norm after the block need a residual")
    if not post and (post_weight is not None or post_bias is not None):
        raise RuntimeError("post_weight and post_bias need post_norm=True")
    w, kw, dt = _param(weight, hidden, dev, None, "weight")
    b, kb, dt = _param(bias, hidden, dev, dt, "bias")
    pw = pb = 0
    if post:
        pw, kpw, dt = _param(post_weight, hidden, dev, dt, "post_weight")
        pb, kpb, dt = _param(post_bias, hidden, dev, dt, "post_bias")
    g = g_code = g_token = g_channel = 0
    if gate is not None:
        if gate.device != dev or gate.dtype not in codes:
            raise RuntimeError(f"gate must be float32, float16 or bfloat16 on {dev}, got "
                               f"{gate.dtype} on {gate.device}")
        try:
            gate = gate.expand(shape)
        except RuntimeError:
            raise RuntimeError(f"gate must broadcast to x's shape {tuple(shape)}, got "
                               f"{tuple(gate.shape)}") from None
        if tokens and hidden:
            gate = gate if gate.dim() == 2 else gate.reshape(-1, hidden)
            if gate.stride(1) not in (0, 1):
                gate = gate.contiguous()
            g, g_code = gate.data_ptr(), codes[gate.dtype]
            g_token, g_channel = gate.stride(0), gate.stride(1) if hidden > 1 else 0
    out = scale = None
    if dtype is not None:
        out = x.new_empty((tokens, hidden), dtype=dtype)
        if dtype is torch.int8:
            scale = x.new_empty((tokens,), dtype=torch.float32)
    if tokens == 0 or hidden == 0:
        return h, out, scale if scale is None else scale.zero_()
    x2, x_stride = _rows(x, hidden)
    r2, r_stride = (None, 0) if residual is None else _rows(residual, hidden)
    args = _ARGS.pack(
        tokens, hidden, x2.data_ptr(), x_stride, 0 if r2 is None else r2.data_ptr(), r_stride, g,
        g_token, g_channel, pw, pb, w, b, 0 if h is None else h.data_ptr(),
        0 if out is None else out.data_ptr(), 0 if scale is None else scale.data_ptr(), code, r_code,
        0 if dt is None else codes[dt], g_code, out_code, k, bool(post), eps, alpha)
    with _abi.on_device(dev):
        rc = _abi.lib().cbq_norm(args, _abi.stream_handle(dev))
    _abi.check(rc, "norm")
    return h, out, scale
