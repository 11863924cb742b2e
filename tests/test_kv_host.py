"""The key/value cache's refusals (no GPU work): C entries and bindings."""
from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]


def _L():
    from cublade_amd import _abi
    return _abi, _abi.lib()


def test_header_and_signatures_agree():
    _abi, L = _L()
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "cublade_kv.h").read_text(), flags=re.S)
    names = set(re.findall(r"\b(cbq_kv_\w+)\s*\(", text))
    assert names == set(_abi.KV_SIGNATURES) and all(hasattr(L, n) for n in names)


def _cache(**kw):
    from cublade_amd import _abi
    f = dict(k=4096, v=4096, k_scale=4096, v_scale=4096, num_pages=4, kv_heads=2, head_dim=64,
             page_size=16, store=0)
    f.update(kw)
    return _abi.KvCache(*[f[n] for n, _ in _abi.KvCache._fields_])


def _batch(**kw):
    from cublade_amd import _abi
    f = dict(page_table=4096, table_stride=4, lengths=4096, cu=None, tokens=2, batch=2, max_pages=4)
    f.update(kw)
    return _abi.KvBatch(*[f[n] for n, _ in _abi.KvBatch._fields_])


def _heads(data=4096, ts=256, hs=64):
    from cublade_amd import _abi
    return _abi.KvHeads(data, ts, hs)


def _refused(rc, needle):
    _, L = _L()
    assert rc == 1 and needle in L.cbq_last_error().decode(), L.cbq_last_error()


def test_c_entries_refuse_bad_arguments():
    _abi, L = _L()
    by = ctypes.byref

    def append(cache=None, batch=None, dtype=1, k=None, v=None, q=None, hq=0, rope=None, out=None):
        return L.cbq_kv_append(by(cache or _cache()), by(batch or _batch()), dtype,
                               by(k or _heads()), by(v or _heads()), by(q) if q else None, hq,
                               by(rope) if rope else None, out, None)

    def attend(cache=None, batch=None, dtype=1, q=None, hq=4, causal=1, window=0, ws=None, n=0,
               out=4096):
        return L.cbq_kv_attend(by(cache or _cache()), by(batch or _batch()), dtype,
                               by(q or _heads()), hq, 1.0, causal, window, 0, ws, n, out, None, None)

    for call in (append, attend):
        _refused(call(cache=_cache(store=2)), "store")
        for d in (0, 8, 72, 272):
            _refused(call(cache=_cache(head_dim=d)), "head_dim")
        for p in (0, 8, 48, 512):
            _refused(call(cache=_cache(page_size=p)), "page_size")
        _refused(call(cache=_cache(kv_heads=0)), "kv_heads")
        _refused(call(cache=_cache(num_pages=-1)), "num_pages")
        _refused(call(cache=_cache(num_pages=1 << 31)), "num_pages")
        _refused(call(cache=_cache(k=None)), "null")
        _refused(call(cache=_cache(v=4104)), "aligned")
        _refused(call(batch=_batch(tokens=3)), "one new token")
        _refused(call(batch=_batch(tokens=-1)), "negative")
        _refused(call(batch=_batch(lengths=None)), "lengths")
        _refused(call(batch=_batch(page_table=None)), "page_table")
        _refused(call(batch=_batch(table_stride=3)), "table_stride")
        _refused(call(dtype=0), "dtype")
        assert call(batch=_batch(tokens=0, batch=0, lengths=None, page_table=None)) == 0
    _refused(append(k=_heads(data=None)), "null k")
    _refused(append(v=_heads(ts=12)), "v must be")
    _refused(append(q=_heads(hs=4), hq=4, out=4096), "q must be")
    _refused(append(q=_heads(), hq=4), "q_out")
    for rot in (3, 66, -2):
        _refused(append(rope=_abi.KvRope(4096, 4096, None, 10, rot, 0)), "rot_dim")
    _refused(append(rope=_abi.KvRope(None, 4096, None, 10, 32, 0)), "null rotation")
    _refused(append(rope=_abi.KvRope(4100, 4096, None, 10, 32, 0)), "aligned")
    _refused(attend(hq=3), "q_heads")
    _refused(attend(hq=0), "q_heads")
    _refused(attend(window=-1), "window")
    _refused(attend(window=4, causal=0), "window")
    _refused(attend(q=_heads(data=4100)), "q must be")
    _refused(attend(out=None), "out")
    _refused(attend(ws=4112, n=1 << 20), "workspace")

    def dequant(cache=None, pages=4096, n=1, k=4096, v=4096, dtype=1):
        return L.cbq_kv_dequant(by(cache or _cache()), pages, n, k, v, dtype, None)

    _refused(dequant(dtype=0), "out_dtype")
    _refused(dequant(n=-1), "negative")
    _refused(dequant(pages=None), "null")
    _refused(dequant(k=4100), "aligned")
    _refused(dequant(cache=_cache(num_pages=0)), "no pages")
    assert dequant(n=0, pages=None) == 0


def test_workspace_query_needs_no_device():
    _abi, L = _L()
    by = ctypes.byref
    c = _abi.WS_CTRL_BYTES
    # enough rows: nothing is split
    assert L.cbq_kv_attend_ws_bytes(by(_cache(kv_heads=8)), by(_batch(tokens=512, batch=512)), 8, 0) == c
    # one short sequence: one range of keys
    assert L.cbq_kv_attend_ws_bytes(by(_cache()), by(_batch(tokens=1, batch=1)), 4, 0) == c
    one = _batch(tokens=1, batch=1, max_pages=8192, table_stride=8192)
    full = L.cbq_kv_attend_ws_bytes(by(_cache()), by(one), 4, 0)
    # at most 64 ranges of the keys, for 2 kv heads a tile of 16 rows of 64 + 2 numbers
    assert c < full <= c + 64 * 2 * 16 * 66 * 4
    assert L.cbq_kv_attend_ws_bytes(by(_cache()), by(one), 4, 256) == c
    assert L.cbq_kv_attend_ws_bytes(by(_cache()), by(one), 3, 0) == c     # refused by the call


def test_bindings_refuse_before_any_device_work():
    from cublade_amd.quantization import QuantizedKVCache
    z = torch.zeros
    good = dict(k=z(2, 1, 16, 32, dtype=torch.int8), v=z(2, 1, 32, 16, dtype=torch.int8),
                k_scale=z(2, 1), v_scale=z(2, 1))
    with pytest.raises(RuntimeError, match="CUDA"):
        QuantizedKVCache(**good)
    for name, t, what in (("k", z(2, 1, 16, 32), "codes"), ("k", z(2, 16, 32, dtype=torch.int8), "4-D"),
                          ("v", z(2, 1, 16, 32, dtype=torch.int8), "v must be"),
                          ("v", z(2, 1, 32, 16).to(torch.float8_e4m3fn), "one dtype"),
                          ("k_scale", z(2, 2), "k_scale"), ("v_scale", z(2, 1).half(), "v_scale")):
        with pytest.raises(RuntimeError, match=what):
            QuantizedKVCache(**{**good, name: t})
    with pytest.raises(ValueError, match="CUDA"):
        QuantizedKVCache.empty(1, 1, 32, device="cpu")
    with pytest.raises(ValueError, match="dtype"):
        QuantizedKVCache.empty(1, 1, 32, dtype=torch.int32)


@pytest.mark.gpu
def test_bindings_refuse_bad_tensors():
    from cublade_amd.quantization import QuantizedKVCache, append_kv, attend_kv, dequantize_kv
    for args in ((2, 1, 24), (2, 1, 512), (2, 1, 32, 24)):
        with pytest.raises(RuntimeError, match="head_dim|page_size"):
            QuantizedKVCache.empty(*args)
    cache = QuantizedKVCache.empty(2, 2, 32, 16)
    with pytest.raises(AttributeError):
        cache.k = cache.v
    import copy
    other = copy.deepcopy(cache)
    assert other.k.data_ptr() != cache.k.data_ptr() and other._view.k == other.k.data_ptr()
    dev = "cuda"
    table = torch.zeros(1, 1, dtype=torch.int32, device=dev)
    n = torch.ones(1, dtype=torch.int32, device=dev)
    x = torch.zeros(1, 2, 32, dtype=torch.float16, device=dev)
    c32 = torch.zeros(4, 16, device=dev)

    def bad(what, fn, *a, **kw):
        with pytest.raises(RuntimeError, match=what):
            fn(*a, **kw)

    bad("k must be", append_kv, cache, x[:, :1], x, table, n)
    bad("v must be", append_kv, cache, x, x.float(), table, n)
    bad("v must be", append_kv, cache, x, x.bfloat16(), table, n)
    bad("k must be", append_kv, cache, x.float(), x, table, n)
    bad("k must be", append_kv, cache, x.cpu(), x, table, n)
    bad("q must be", append_kv, cache, x, x, table, n, q=x[..., :16])
    bad("page_table", append_kv, cache, x, x, table.long(), n)
    bad("page_table", append_kv, cache, x, x, table[0], n)
    bad("lengths", append_kv, cache, x, x, table, n.cpu())
    bad("lengths", append_kv, cache, x, x, table, n.repeat(2))
    bad("one new token", append_kv, cache, x.repeat(2, 1, 1), x.repeat(2, 1, 1), table, n)
    bad("offsets", append_kv, cache, x, x, table, n, cu_new=n)
    bad("no sequence", append_kv, cache, x, x, table[:0], n[:0], cu_new=n)
    bad("rope", append_kv, cache, x, x, table, n, rope=(c32.half(), c32))
    bad("rope", append_kv, cache, x, x, table, n, rope=(c32, c32[:2]))
    bad("rope", append_kv, cache, x, x, table, n, rope=(c32.repeat(1, 2), c32.repeat(1, 2)))
    bad("positions", append_kv, cache, x, x, table, n, rope=(c32, c32), positions=n)
    bad("positions", append_kv, cache, x, x, table, n, positions=n.long())
    bad("heads", attend_kv, x[:, :1], cache, table, n)
    bad("q must be", attend_kv, x[0], cache, table, n)
    bad("window", attend_kv, x, cache, table, n, window=0)
    bad("window", attend_kv, x, cache, table, n, window=3, causal=False)
    bad("max_length", attend_kv, x, cache, table, n, max_length=-1)
    bad("pages", dequantize_kv, cache, table)
    bad("out_dtype", dequantize_kv, cache, n, torch.float32)
