"""8-bit paged key/value cache on the HIP C ABI (include/cublade_kv.h): append
with position rotation, attention, read-back. No counterpart in the reference.

Every function takes the cache as its ctypes view (_abi.KvCache, made by
kv_cache_view) and launches on the current stream of the cache's device. What
the kernels find in page tables, lengths and offsets on the device is bounded
there, not here: nothing synchronises.
"""
from __future__ import annotations

import ctypes
import math

import torch

from ... import _abi
from ._common import out_like

STORE_CODE = {torch.int8: _abi.KV_INT8, torch.float8_e4m3fn: _abi.KV_FP8}
_DTYPES = (torch.float16, torch.bfloat16)


def kv_cache_view(k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor,
                  v_scale: torch.Tensor) -> _abi.KvCache:
    """The ctypes view of a cache's tensors (which the caller keeps alive):
    k [num_pages, kv_heads, page_size, head_dim] and v [num_pages, kv_heads,
    head_dim, page_size], int8 or float8_e4m3fn; scales [num_pages, kv_heads]
    float32."""
    if k.dtype not in STORE_CODE:
        raise RuntimeError(f"kv cache: codes must be torch.int8 or torch.float8_e4m3fn, got {k.dtype}")
    if k.dim() != 4 or v.dim() != 4 or v.dtype != k.dtype:
        raise RuntimeError("kv cache: k and v must be 4-D and of one dtype")
    pages, heads, page, d = k.shape
    if tuple(v.shape) != (pages, heads, d, page):
        raise RuntimeError(f"kv cache: v must be [pages, heads, head_dim, page_size] = "
                           f"{(pages, heads, d, page)}, got {tuple(v.shape)}")
    for t, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
        if t.dtype != torch.float32 or tuple(t.shape) != (pages, heads):
            raise RuntimeError(f"kv cache: {name} must be float32 [{pages}, {heads}], got "
                               f"{t.dtype} {tuple(t.shape)}")
    for t in (k, v, k_scale, v_scale):
        if not t.is_cuda or t.device != k.device:
            raise RuntimeError("kv cache: all tensors must be on one CUDA device")
        if not t.is_contiguous():
            raise RuntimeError("kv cache: all tensors must be contiguous")
    if d % 16 or not 16 <= d <= 256:
        raise RuntimeError(f"kv cache: head_dim must be a multiple of 16 in [16, 256], got {d}")
    if page not in (16, 32, 64, 128, 256):
        raise RuntimeError(f"kv cache: page_size must be 16, 32, 64, 128 or 256, got {page}")
    return _abi.KvCache(_abi.ptr(k), _abi.ptr(v), _abi.ptr(k_scale), _abi.ptr(v_scale), pages,
                        heads, d, page, STORE_CODE[k.dtype])


def _index(t: torch.Tensor, dev: torch.device, dims: int, name: str) -> None:
    if t.dtype != torch.int32 or t.dim() != dims or t.device != dev:
        raise RuntimeError(f"{name} must be a {dims}-D torch.int32 tensor on {dev}, got "
                           f"{t.dim()}-D {t.dtype} on {t.device}")


def _batch(dev, tokens: int, page_table, lengths, cu):
    """(KvBatch, tensors it points to)."""
    _index(page_table, dev, 2, "page_table")
    _index(lengths, dev, 1, "lengths")
    batch, width = page_table.shape
    if lengths.numel() != batch:
        raise RuntimeError(f"lengths must have {batch} elements, one per row of page_table, got "
                           f"{lengths.numel()}")
    if width > 1 and page_table.stride(1) != 1:
        page_table = page_table.contiguous()
    if not lengths.is_contiguous():
        lengths = lengths.contiguous()
    stride = page_table.stride(0) if batch > 1 else width
    if cu is None:
        if tokens != batch:
            raise RuntimeError(f"without offsets each of the {batch} sequences has one new token, "
                               f"got {tokens} tokens")
        cu_ptr = None
    else:
        _index(cu, dev, 1, "the offsets of new tokens")
        if cu.numel() != batch + 1:
            raise RuntimeError(f"the offsets of new tokens must have {batch + 1} elements, got "
                               f"{cu.numel()}")
        if not cu.is_contiguous():
            cu = cu.contiguous()
        cu_ptr = cu.data_ptr()
        if batch == 0 and tokens:
            raise RuntimeError(f"{tokens} tokens of no sequence")
    if stride < width:      # an expanded table
        page_table = page_table.contiguous()
        stride = width
    return (_abi.KvBatch(page_table.data_ptr(), stride, lengths.data_ptr(), cu_ptr, tokens, batch,
                         width), (page_table, lengths, cu))


def _heads(x: torch.Tensor, dev, dtype, heads: int | None, d: int, tokens: int | None, name: str):
    """(KvHeads, the tensor it points to): x as it is where the kernels can
    read its strides, else a contiguous copy."""
    if x.dim() != 3 or x.size(2) != d or (heads is not None and x.size(1) != heads) or (
            tokens is not None and x.size(0) != tokens):
        raise RuntimeError(f"{name} must be [{'tokens' if tokens is None else tokens}, "
                           f"{'heads' if heads is None else heads}, {d}], got {tuple(x.shape)}")
    if x.device != dev:
        raise RuntimeError(f"{name} must be on the cache's device {dev}, got {x.device}")
    if x.dtype not in _DTYPES or (dtype is not None and x.dtype != dtype):
        want = "torch.float16 or torch.bfloat16" if dtype is None else str(dtype)
        raise RuntimeError(f"{name} must be {want}, got {x.dtype}")
    ts, hs, es = x.stride()
    p = x.data_ptr()
    if es != 1 or ts % 8 or hs % 8 or p % 16:
        x = x.clone(memory_format=torch.contiguous_format)
        ts, hs, _ = x.stride()
        p = x.data_ptr()
    return _abi.KvHeads(p, ts, hs), x


def kv_append(view: _abi.KvCache, dev: torch.device, k: torch.Tensor, v: torch.Tensor,
              page_table: torch.Tensor, lengths: torch.Tensor,
              cu_new: torch.Tensor | None = None,
              rope: tuple[torch.Tensor, torch.Tensor] | None = None, interleaved: bool = False,
              positions: torch.Tensor | None = None,
              q: torch.Tensor | None = None) -> torch.Tensor | None:
    """Rotate and append new keys and values, rotate the queries; see
    quantization.kv_cache.append_kv."""
    heads, d = view.kv_heads, view.head_dim
    ck, k = _heads(k, dev, None, heads, d, None, "k")
    tokens, dt = k.size(0), k.dtype
    cv, v = _heads(v, dev, dt, heads, d, tokens, "v")
    batch, keep = _batch(dev, tokens, page_table, lengths, cu_new)
    cq = out = None
    hq = 0
    if q is not None:
        cq, q = _heads(q, dev, dt, None, d, tokens, "q")
        hq = q.size(1)
        out = out_like(q, dt)
    cr = None
    if rope is not None:
        cos, sin = rope
        if cos.dtype != torch.float32 or sin.dtype != torch.float32 or cos.dim() != 2 or \
                cos.shape != sin.shape or cos.device != dev or sin.device != dev:
            raise RuntimeError(f"rope must be two float32 [rows, rot_dim / 2] tensors on {dev}")
        rot = 2 * cos.size(1)
        if rot > d:
            raise RuntimeError(f"rope turns {rot} dimensions of heads of {d}")
        cos = cos if cos.is_contiguous() and cos.data_ptr() % 16 == 0 else cos.clone(
            memory_format=torch.contiguous_format)
        sin = sin if sin.is_contiguous() and sin.data_ptr() % 16 == 0 else sin.clone(
            memory_format=torch.contiguous_format)
        pp = None
        if positions is not None:
            if positions.dtype != torch.int64 or tuple(positions.shape) != (tokens,) or \
                    positions.device != dev:
                raise RuntimeError(f"positions must be a torch.int64 [{tokens}] tensor on {dev}")
            positions = positions.contiguous()
            pp = positions.data_ptr()
        cr = _abi.KvRope(cos.data_ptr(), sin.data_ptr(), pp, cos.size(0), rot, bool(interleaved))
    elif positions is not None:
        raise RuntimeError("positions are given without rope")
    if tokens == 0:
        return out
    by = ctypes.byref
    with _abi.on_device(dev):
        rc = _abi.lib().cbq_kv_append(by(view), by(batch), _abi.DTYPE_CODE[dt], by(ck), by(cv),
                                      by(cq) if cq is not None else None, hq,
                                      by(cr) if cr is not None else None, _abi.ptr(out),
                                      _abi.stream_handle(dev))
    _abi.check(rc, "append_kv")
    return out


def kv_dequantize(view: _abi.KvCache, dev: torch.device, pages: torch.Tensor,
                  out_dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    """Pages read back as 16-bit values; see quantization.kv_cache.dequantize_kv."""
    _index(pages, dev, 1, "pages")
    if out_dtype not in _DTYPES:
        raise RuntimeError("out_dtype must be torch.float16 or torch.bfloat16")
    pages = pages.contiguous()
    n = pages.numel()
    shape = (n, view.kv_heads, view.page_size, view.head_dim)
    k = torch.empty(shape, dtype=out_dtype, device=dev)
    v = torch.empty(shape, dtype=out_dtype, device=dev)
    if n == 0:
        return k, v
    with _abi.on_device(dev):
        rc = _abi.lib().cbq_kv_dequant(ctypes.byref(view), pages.data_ptr(), n, k.data_ptr(),
                                       v.data_ptr(), _abi.DTYPE_CODE[out_dtype],
                                       _abi.stream_handle(dev))
    _abi.check(rc, "dequantize_kv")
    return k, v


def kv_attend(view: _abi.KvCache, dev: torch.device, q: torch.Tensor, page_table: torch.Tensor,
              lengths: torch.Tensor, cu_q: torch.Tensor | None = None,
              scale: float | None = None, causal: bool = True, window: int | None = None,
              max_length: int | None = None, return_lse: bool = False):
    """Attention over the cache; see quantization.kv_cache.attend_kv."""
    cq, q = _heads(q, dev, None, None, view.head_dim, None, "q")
    tokens, hq, d = q.shape
    if hq == 0 or hq % view.kv_heads:
        raise RuntimeError(f"q must have a positive multiple of {view.kv_heads} heads, got {hq}")
    if window is not None and (window <= 0 or not causal):
        raise RuntimeError(f"window must be positive and needs causal=True, got {window}")
    if max_length is not None and max_length < 0:
        raise RuntimeError(f"max_length must not be negative, got {max_length}")
    batch, keep = _batch(dev, tokens, page_table, lengths, cu_q)
    out = out_like(q, q.dtype)
    lse = torch.empty((tokens, hq), dtype=torch.float32, device=dev) if return_lse else None
    if tokens:
        L = _abi.lib()
        by = ctypes.byref
        ml = max_length or 0
        with _abi.on_device(dev), _abi.workspace_lock(dev):
            ws = _abi.workspace(dev, L.cbq_kv_attend_ws_bytes(by(view), by(batch), hq, ml))
            rc = L.cbq_kv_attend(by(view), by(batch), _abi.DTYPE_CODE[q.dtype], by(cq), hq,
                                 1.0 / math.sqrt(d) if scale is None else float(scale), bool(causal),
                                 window or 0, ml, ws.data_ptr(), ws.numel(), out.data_ptr(),
                                 _abi.ptr(lse), _abi.stream_handle(dev))
        _abi.check(rc, "attend_kv")
    return (out, lse) if return_lse else out
