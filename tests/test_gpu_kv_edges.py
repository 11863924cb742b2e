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
