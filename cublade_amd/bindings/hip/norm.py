"""The norms before and after a block on the HIP C ABI (include/cublade_w8a8.h).
No counterpart in the reference."""
from __future__ import annotations

import ctypes
import math

import torch

from ... import _abi


def _rows(x: torch.Tensor, hidden: int) -> tuple[torch.Tensor, int]:
    """x (not empty) as [tokens, hidden] whose rows the kernel can read in place,
    and the elements from one row to the next."""
    x2 = x if x.dim() == 2 else x.reshape(-1, hidden)
    if x2.size(0) > 1 and x2.stride(0) < hidden or hidden > 1 and x2.stride(1) != 1:
        x2 = x2.contiguous()
    return x2, x2.stride(0) if x2.size(0) > 1 else hidden


def _param(p: torch.Tensor | None, hidden: int, dev: torch.device, dtype, name: str):
    """(data pointer or None, the tensor it points to, the parameters' dtype)."""
    if p is None:
        return None, None, dtype
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
    code = _abi.DTYPE_CODE.get(x.dtype)
    if code is None:
        raise RuntimeError(f"x must be float32, float16 or bfloat16, got {x.dtype}")
    if x.dim() < 1:
        raise RuntimeError("x must have at least 1 dimension")
    k = _abi.NORM_CODE.get(kind)
    if k is None:
        raise RuntimeError(f"kind must be one of {sorted(_abi.NORM_CODE)}, got {kind!r}")
    dev, shape, hidden = x.device, x.shape, x.shape[-1]
    out_code = _abi.I8 if dtype is torch.int8 else _abi.DTYPE_CODE.get(dtype)
    if out_code is None:
        if dtype is not None:
            raise RuntimeError(f"dtype must be int8, float32, float16 or bfloat16, got {dtype}")
        out_code = 0
    tokens = math.prod(shape[:-1])
    h = None
    r_code = code
    if residual is not None:
        if residual.shape != shape or residual.device != dev or (
                residual.dtype != x.dtype and residual.dtype != torch.float32):
            raise RuntimeError(f"residual must be {tuple(shape)} in x's dtype or float32 on {dev}, "
                               f"got {tuple(residual.shape)} {residual.dtype} on {residual.device}")
        r_code = _abi.DTYPE_CODE[residual.dtype]
        h = torch.empty(shape, dtype=residual.dtype, device=dev)
    elif post or gate is not None:
        raise RuntimeError("a gate and a norm after the block need a residual")
    if not post and (post_weight is not None or post_bias is not None):
        raise RuntimeError("post_weight and post_bias need post_norm=True")
    w, kw, dt = _param(weight, hidden, dev, None, "weight")
    b, kb, dt = _param(bias, hidden, dev, dt, "bias")
    pw, kpw, dt = _param(post_weight, hidden, dev, dt, "post_weight")
    pb, kpb, dt = _param(post_bias, hidden, dev, dt, "post_bias")
    g, g_code, g_token, g_channel = None, 0, 0, 0
    if gate is not None:
        if gate.device != dev or gate.dtype not in _abi.DTYPE_CODE:
            raise RuntimeError(f"gate must be float32, float16 or bfloat16 on {dev}, got "
                               f"{gate.dtype} on {gate.device}")
        try:
            gate = gate.expand(shape)
        except RuntimeError:
            raise RuntimeError(f"gate must broadcast to x's shape {tuple(shape)}, got "
                               f"{tuple(gate.shape)}") from None
        if x.numel():
            gate = gate if gate.dim() == 2 else gate.reshape(-1, hidden)
            if gate.stride(1) not in (0, 1):
                gate = gate.contiguous()
            g, g_code = gate.data_ptr(), _abi.DTYPE_CODE[gate.dtype]
            g_token, g_channel = gate.stride(0), gate.stride(1) if hidden > 1 else 0
    out = scale = None
    if dtype is not None:
        out = torch.empty((tokens, hidden), dtype=dtype, device=dev)
        if out_code == _abi.I8:
            scale = torch.empty((tokens,), dtype=torch.float32, device=dev)
    if x.numel() == 0:
        return h, out, scale if scale is None else scale.zero_()
    x2, x_stride = _rows(x, hidden)
    r2, r_stride = (None, 0) if residual is None else _rows(residual, hidden)
    args = _abi.NormArgs(
        tokens, hidden, x2.data_ptr(), x_stride, _abi.ptr(r2), r_stride, g, g_token, g_channel, pw, pb,
        w, b, _abi.ptr(h), _abi.ptr(out), _abi.ptr(scale), code, r_code,
        0 if dt is None else _abi.DTYPE_CODE[dt], g_code, out_code, k, bool(post), eps, alpha)
    with _abi.on_device(dev):
        rc = _abi.lib().cbq_norm(ctypes.byref(args), _abi.stream_handle(dev))
    _abi.check(rc, "norm")
    return h, out, scale
