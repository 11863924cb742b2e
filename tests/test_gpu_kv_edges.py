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


def _poison(q):
    """Leaves NaN in the allocator's next free block of q's size and its lse's."""
    for shape, dt in ((q.shape, q.dtype), (q.shape[:2], torch.float32)):
        t = torch.full(shape, math.nan, dtype=dt, device=DEV)
        del t


PADDED = [
    # kv heads, heads of each, d, lens, news, tokens in front and behind, window
    (2, 4, 64, [40, 90, 7], [1, 3, 0], 0, 5, None),
    (2, 4, 64, [40, 90, 7], [1, 3, 0], 2, 0, None),
    (1, 8, 128, [9000], [5], 3, 60, None),
    (2, 4, 128, [300], [200], 1, 300, None),
    (1, 2, 80, [400, 50, 9], [300, 1, 1], 7, 70, None),
    (2, 4, 64, [400, 50, 9], [100, 1, 1], 7, 70, 40),
    (1, 1, 256, [3, 2], [0, 0], 0, 4, None),
]


@pytest.mark.parametrize("store,dt", [(I8, BF16), (F8, F16)])
@pytest.mark.parametrize("case", range(len(PADDED)))
def test_tokens_of_no_sequence_are_zero(case, store, dt):
    """Tokens in front of the first offset and behind the last (a batch padded
    to a fixed size): zeros and -infinity, and the others as without them."""
    from cublade_amd.quantization import attend_kv
    hkv, rep, d, lens, news, front, behind, window = PADDED[case]
    g = _gen(60 + case)
    table, pages = _kv.make_table(lens, 32, g)
    cache = _kv.random_cache(pages, hkv, d, 32, store, g)
    t = sum(news)
    q = torch.randn(front + t + behind, hkv * rep, d, generator=g, device=DEV).to(dt)
    cu = _cu(news) + front
    _poison(q)
    o, lse = attend_kv(q, cache, table, _i32(lens), cu_q=cu, window=window, return_lse=True)
    own = slice(front, front + t)
    ref = _kv.attend_ref(q[own], cache, table, lens, news, window=window)
    _kv.assert_attends((o[own], lse[own]), ref, dt, PADDED[case])
    rest = torch.ones(q.shape[0], dtype=torch.bool, device=DEV)
    rest[own] = False
    assert bool((o[rest] == 0).all()) and bool((lse[rest] == -math.inf).all())


def test_appended_queries_of_no_sequence_have_no_position():
    """Queries in front of the first offset and behind the last: NaN where they
    would be rotated, whatever stands at the sequences' positions; unless each
    token's row is given."""
    from cublade_amd.quantization import append_kv
    g = _gen(70)
    lens, news, front, behind = [40, 90], [3, 2], 2, 4
    table, pages = _kv.make_table(lens, 16, g)
    cache = _kv.random_cache(pages, 2, 64, 16, I8, g)
    model = _kv.CacheModel(cache)
    x = torch.randn(11, 2, 64, generator=g, device=DEV).half()
    rope = _kv.tables(100, 32)
    own = slice(front, front + 5)
    pos = torch.tensor([37, 38, 39, 88, 89], device=DEV)
    out = append_kv(cache, x, x, table, _i32(lens), cu_new=_cu(news) + front, rope=rope, q=x)
    turned = _kv.rotate_f32(x[own], pos, *rope, False)
    assert torch.equal(out[own], turned.half())
    rest = [0, 1, 7, 8, 9, 10]
    assert bool(out[rest][..., :32].isnan().all()) and torch.equal(out[rest][..., 32:], x[rest][..., 32:])
    model.append(turned, x[own], table, lens, news)
    model.assert_equal(cache)
    every = torch.arange(11, device=DEV)
    out = append_kv(cache, x, x, table, _i32(lens), cu_new=_cu(news) + front, rope=rope, q=x,
                    positions=every)
    assert torch.equal(out, _kv.rotate_f32(x, every, *rope, False).half())


def test_padded_batch_replayed_from_a_graph():
    """One captured call of a fixed number of tokens, replayed for batches that
    bring fewer: each replay as the eager call, eager work between them."""
    from cublade_amd.quantization import attend_kv
    g = _gen(71)
    lens = [500, 300, 40]
    table, pages = _kv.make_table(lens, 16, g)
    cache = _kv.random_cache(pages, 2, 64, 16, I8, g)
    q = torch.randn(240, 8, 64, generator=g, device=DEV).bfloat16()
    n, cu = _i32(lens), _cu([1, 1, 1])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        attend_kv(q, cache, table, n, cu_q=cu, return_lse=True)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            o, lse = attend_kv(q, cache, table, n, cu_q=cu, return_lse=True)
        for news in ([1, 1, 1], [200, 30, 10], [0, 0, 0], [1, 100, 1], [1, 1, 1]):
            cu.copy_(_cu(news))
            o.fill_(math.nan)
            lse.fill_(math.nan)
            graph.replay()
            s.synchronize()
            eager = attend_kv(q, cache, table, n, cu_q=cu, return_lse=True)
            assert torch.equal(o, eager[0]) and torch.equal(lse, eager[1])
            assert bool((o[sum(news):] == 0).all()) and bool(o[:sum(news)].isfinite().all())
