"""More refusals of the key/value cache's C entries (no GPU work)."""
from __future__ import annotations

import ctypes


def test_append_refuses_negative_query_heads():
    from cublade_amd import _abi
    L, by = _abi.lib(), ctypes.byref
    cache = _abi.KvCache(4096, 4096, 4096, 4096, 4, 2, 64, 16, _abi.KV_INT8)
    # no token: nothing is launched, whatever is refused
    batch = _abi.KvBatch(4096, 4, 4096, None, 0, 0, 4)
    heads = _abi.KvHeads(4096, 256, 64)

    def append(q, q_heads):
        return L.cbq_kv_append(by(cache), by(batch), _abi.F16, by(heads), by(heads),
                               by(heads) if q else None, q_heads, None, 4096, None)

    assert append(True, 4) == 0 and append(True, 0) == 0 and append(False, 0) == 0
    for q in (True, False):
        assert append(q, -1) == 1 and b"q_heads" in L.cbq_last_error()
