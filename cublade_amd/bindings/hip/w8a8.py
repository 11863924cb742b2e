"""Products of INT8 activations and INT8 weights on the HIP C ABI
(include/cublade_w8a8.h). No counterpart in the reference."""
from __future__ import annotations

import ctypes
import functools

import torch

from ... import _abi

_MAX_STRIDE = 1 << 22      # bytes between rows that the kernels take


def _rows(codes: torch.Tensor, scale: torch.Tensor, dev: torch.device, k: int | None, name: str):
    """(I8Rows, rows, columns, the tensors it points to): codes as they are where
    the kernels can read their rows, else a contiguous copy."""
    shape = codes.shape
    if codes.dtype is not torch.int8 or len(shape) != 2 or (k is not None and shape[1] != k):
        raise RuntimeError(f"{name} must be int8 [rows, {'columns' if k is None else k}], got "
                           f"{tuple(shape)} {codes.dtype}")
    if codes.device != dev or scale.device != dev:
        raise RuntimeError(f"{name} and its scales must be on {dev}, got {codes.device} and "
                           f"{scale.device}")
    if scale.dtype is not torch.float32:
        raise RuntimeError(f"{name} must have torch.float32 scales, got {scale.dtype}")
    rows, cols = shape
    step = scale.dim()
    if step:
        if step != 1 or scale.numel() != rows:
            raise RuntimeError(f"{name} must have one scale for each of its {rows} rows, or a 0-d "
                               f"one for all, got {tuple(scale.shape)}")
        if not scale.is_contiguous():
            scale = scale.contiguous()
    stride, es = codes.stride()
    p = codes.data_ptr()
    if es != 1 or stride < cols or stride > _MAX_STRIDE or (cols % 16 == 0 and (stride % 16 or p % 16)):
        codes = codes.clone(memory_format=torch.contiguous_format)
        stride, p = cols, codes.data_ptr()
    return _abi.I8Rows(p, stride, scale.data_ptr(), step), rows, cols, (codes, scale)


def _bias(b: torch.Tensor | None, n: int, dev: torch.device, name: str):
    if b is None:
        return None
    if b.device != dev or b.dtype not in _abi.DTYPE_CODE or b.dim() != 1 or b.numel() != n:
        raise RuntimeError(f"{name} must be [{n}] in float32, float16 or bfloat16 on {dev}, got "
                           f"{tuple(b.shape)} {b.dtype} on {b.device}")
    return b.detach().contiguous()


def _out_code(dtype: torch.dtype) -> int:
    code = _abi.DTYPE_CODE.get(dtype)
    if code is None:
        raise RuntimeError(f"out_dtype must be float32, float16 or bfloat16, got {dtype}")
    return code


def _check_cuda(x: torch.Tensor, what: str) -> None:
    if not x.is_cuda:
        raise RuntimeError(f"{what}: x must be on CUDA, got {x.device}")


@functools.lru_cache(maxsize=4096)
def _ws_bytes(device: int | None, m: int, n: int, k: int, projections: int) -> int:
    """Workspace of a call on the current device, by its sizes alone."""
    return _abi.lib().cbq_w8a8_ws_bytes(m, n, k, projections)


def _run(call, args, dev: torch.device, size, what: str) -> None:
    with _abi.on_device(dev):
        need = _ws_bytes(dev.index, *size)
        if need <= _abi.WS_CTRL_BYTES:      # one launch that passes nothing on
            rc = call(*args, None, 0, _abi.stream_handle(dev))
        else:
            with _abi.workspace_lock(dev):
                ws = _abi.workspace(dev, need)
                rc = call(*args, ws.data_ptr(), ws.numel(), _abi.stream_handle(dev))
    _abi.check(rc, what)


def w8a8_linear(x: torch.Tensor, x_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
                bias: torch.Tensor | None, out_dtype: torch.dtype) -> torch.Tensor:
    """y[m, n] = x_scale[m] w_scale[n] sum_k x[m, k] w[n, k] + bias[n]; see
    quantization.w8a8.linear_w8a8."""
    _check_cuda(x, "w8a8_linear")
    dev = x.device
    cx, m, k, keep_x = _rows(x, x_scale, dev, None, "x")
    cw, n, _, keep_w = _rows(w, w_scale, dev, k, "weight")
    b = _bias(bias, n, dev, "bias")
    code = _out_code(out_dtype)
    y = x.new_empty((m, n), dtype=out_dtype)
    if m == 0 or n == 0:
        return y
    call = _abi.lib().cbq_w8a8_linear
    args = (ctypes.byref(cx), ctypes.byref(cw), _abi.ptr(b),
            0 if b is None else _abi.DTYPE_CODE[b.dtype], m, n, k, y.data_ptr(), code)
    _run(call, args, dev, (m, n, k, 1), "w8a8_linear")
    return y


def w8a8_gated(x: torch.Tensor, x_scale: torch.Tensor, gate: torch.Tensor,
               gate_scale: torch.Tensor, up: torch.Tensor, up_scale: torch.Tensor,
               activation: str, gate_bias: torch.Tensor | None, up_bias: torch.Tensor | None,
               out_dtype: torch.dtype) -> torch.Tensor:
    """act(x . gate^T + gate_bias) (x . up^T + up_bias); see
    quantization.w8a8.gated_w8a8."""
    _check_cuda(x, "w8a8_gated")
    act = _abi.ACT_CODE.get(activation)
    if act is None:
        raise RuntimeError(f"activation must be one of {sorted(_abi.ACT_CODE)}, got {activation!r}")
    dev = x.device
    cx, m, k, keep_x = _rows(x, x_scale, dev, None, "x")
    cg, n, _, keep_gate = _rows(gate, gate_scale, dev, k, "gate")
    cu, n_up, _, keep_up = _rows(up, up_scale, dev, k, "up")
    if n_up != n:
        raise RuntimeError(f"gate and up must have equally many rows, got {n} and {n_up}")
    gb, ub = _bias(gate_bias, n, dev, "gate_bias"), _bias(up_bias, n, dev, "up_bias")
    if gb is not None and ub is not None and gb.dtype != ub.dtype:
        raise RuntimeError(f"gate_bias and up_bias must have one dtype, got {gb.dtype} and {ub.dtype}")
    code = _out_code(out_dtype)
    y = x.new_empty((m, n), dtype=out_dtype)
    if m == 0 or n == 0:
        return y
    some = gb if gb is not None else ub
    call = _abi.lib().cbq_w8a8_gated
    args = (ctypes.byref(cx), ctypes.byref(cg), ctypes.byref(cu), _abi.ptr(gb), _abi.ptr(ub),
            0 if some is None else _abi.DTYPE_CODE[some.dtype], act, m, n, k, y.data_ptr(), code)
    _run(call, args, dev, (m, n, k, 2), "w8a8_gated")
    return y
