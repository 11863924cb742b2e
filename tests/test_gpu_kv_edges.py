"""attend_kv and append_kv at the edges of their definitions: rows whose scores
are all infinite, offsets that leave tokens out, heads past 2 GiB of a token."""
from __future__ import annotations

import math

import pytest
import torch

from tests import _kv

pytestmark = pytest.mark.gpu
DEV = "cuda"
I8, F8 = torch.int8, torch.float8_e4m3fn
F16, BF16 = torch.float16, torch.bfloat16


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _cu(news):
    c = [0]
    for n in news:
        c.append(c[-1] + n)
    return _i32(c)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("store", [I8, F8])
@pytest.mark.parametrize("n,new", [(1, None), (70, None), (9000, None), (1, 1), (100, 100), (9000, 100)])
@pytest.mark.parametrize("sign", [1, -1])
def test_rows_of_infinite_scores_are_nan(n, new, store, dt, sign):
    """An infinite query element whose products with every visible key are of
    one sign: the softmax over such scores is NaN, and only a row that sees no
    key is 0. Of scores of -infinity the log-sum-exp is -infinity, as for that
    row. One key, several, keys in ranges (9000), single tokens and prompts."""
    from cublade_amd.quantization import attend_kv
    g = _gen(51)
    lens = [n, n, 0]
    news = [new, new, 1] if new else [1, 1, 1]
    table, pages = _kv.make_table(lens, 16, g)
    cache = _kv.random_cache(pages, 1, 64, 16, store, g)
    cache.k[..., 3] = torch.tensor(5.0, device=DEV).to(store)
    q = torch.randn(sum(news), 2, 64, generator=g, device=DEV).to(dt)
    first = news[0]
    q[:first, 1, 3] = sign * math.inf
    o, lse = attend_kv(q, cache, table, _i32(lens), cu_q=_cu(news) if new else None, return_lse=True)
    assert bool(o[:first, 1].isnan().all())
    if sign < 0:
        assert bool((lse[:first, 1] == -math.inf).all())
    else:
        assert not bool(lse[:first, 1].isfinite().any())
    for x in (o, lse):
        assert bool(x[:first, 0].isfinite().all()) and bool(x[first:-1].isfinite().all())
    assert bool((o[-1] == 0).all()) and bool((lse[-1] == -math.inf).all())


@pytest.mark.parametrize("style", ["none", "half", "interleaved"])
def test_queries_past_2_gib_of_a_token(style):
    """A token's rotated queries of more than 2^31 bytes: the last heads are
    written where they belong."""
    from cublade_amd.quantization import QuantizedKVCache, append_kv
    d, hq = 256, (1 << 22) + 64
    cache = QuantizedKVCache.empty(1, 1, d, 16)
    g = _gen(52)
    q = torch.empty(1, hq, d, dtype=F16, device=DEV)
    q.view(torch.int16).random_(0, 0x7C00, generator=g)     # finite numbers
    k = torch.ones(1, 1, d, device=DEV).half()
    cos, sin = (t[5:6].contiguous() for t in _kv.tables(6, d))
    positions = torch.zeros(1, dtype=torch.int64, device=DEV)
    kw = {} if style == "none" else dict(rope=(cos, sin), interleaved=style == "interleaved",
                                         positions=positions)
    out = append_kv(cache, k, k, _i32([[0]]), _i32([1]), q=q, **kw)
    for part in (slice(0, 64), slice(hq // 2, hq // 2 + 64), slice(hq - 128, hq)):
        want = q[:, part]
        if kw:
            want = _kv.rotate_f32(want, positions, cos, sin, style == "interleaved").half()
        assert torch.equal(out[:, part], want)
    if style == "none":
        assert torch.equal(out, q)
