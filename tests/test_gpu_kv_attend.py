"""attend_kv on the GPU against attention in 64 bits over the same codes and
scales, with the error bound of tests/_kv.py."""
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


def _check(d, page, store, dt, hkv, rep, lens, news=None, seed=0, width=None, spread=1.0, **kw):
    from cublade_amd.quantization import attend_kv
    g = _gen(seed)
    step = news is None
    news = [1] * len(lens) if step else news
    table, pages = _kv.make_table(lens, page, g, width)
    cache = _kv.random_cache(pages, hkv, d, page, store, g, spread)
    q = torch.randn(sum(news), hkv * rep, d, generator=g, device=DEV).to(dt)
    extra = {k: kw.pop(k) for k in ("max_length",) if k in kw}
    got = attend_kv(q, cache, table, _i32(lens), cu_q=None if step else _cu(news), return_lse=True,
                    **kw, **extra)
    ref = _kv.attend_ref(q, cache, table, lens, news, **kw)
    _kv.assert_attends(got, ref, dt, (d, page, store, dt, hkv, rep, lens, news, kw))
    return q, cache, table, got


LENS = [1, 15, 16, 17, 63, 64, 65, 130, 257]


@pytest.mark.parametrize("store,dt", [(I8, BF16), (F8, F16), (I8, F16), (F8, BF16)])
@pytest.mark.parametrize("d,page", [(128, 64), (64, 16), (16, 32), (80, 16), (96, 128), (192, 256),
                                    (256, 32), (240, 64)])
def test_single_tokens(d, page, store, dt):
    _check(d, page, store, dt, 2, 4, LENS)


@pytest.mark.parametrize("rep", [1, 2, 7, 16, 17, 40])
def test_shared_heads(rep):
    _check(64, 32, I8, BF16, 3, rep, [5, 100, 64])


@pytest.mark.parametrize("store,dt", [(I8, BF16), (F8, F16)])
@pytest.mark.parametrize("d,page", [(128, 64), (64, 16), (48, 32), (192, 128), (256, 16)])
def test_several_tokens(d, page, store, dt):
    """Drafted tokens and prompts: one to a few hundred queries, pages and tiles
    that end inside one another, sequences that bring nothing."""
    _check(d, page, store, dt, 2, 3, [1, 40, 64, 200, 333, 129, 70], [1, 3, 0, 17, 333, 100, 70])


@pytest.mark.parametrize("window", [1, 5, 64, 100, 1000])
def test_window(window):
    _check(64, 16, I8, F16, 2, 2, [300, 64, 7, 150], [300, 1, 7, 33], window=window)
    _check(64, 16, F8, F16, 2, 2, [300, 64, 7], window=window)


def test_not_causal():
    _check(128, 32, I8, BF16, 2, 2, [100, 64, 1, 31], [7, 64, 1, 31], causal=False)
    _check(128, 32, F8, BF16, 2, 2, [100, 64, 1], causal=False)


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 4.0])
def test_scale(scale):
    _check(32, 16, I8, F16, 1, 2, [50, 200], [10, 130], scale=scale)


@pytest.mark.parametrize("store", [I8, F8])
def test_long_axis_is_split(store):
    """Few rows over a long context: the keys are cut over workgroups, also with
    max_length and a wider table."""
    for kw in ({}, {"max_length": 9000}, {"width": 2000}):
        _check(128, 64, store, BF16, 2, 4, [9000, 3], **kw)
    _check(64, 16, store, F16, 1, 8, [20001], [5])
    _check(64, 16, store, F16, 1, 8, [20001], [5], window=3000)


def test_long_prompt_chunk():
    _check(128, 64, I8, BF16, 2, 4, [4100], [600])
    _check(64, 128, F8, F16, 1, 1, [2500], [2500])


def test_scales_far_apart():
    """Page scales within 2^-20 .. 2^20 of each other: the weights carry the
    value scales, so none of them may over- or underflow."""
    _check(64, 16, I8, BF16, 2, 2, [400, 100], seed=3, spread=20.0, scale=1e-8)
    _check(64, 16, F8, BF16, 2, 2, [400, 100], [40, 100], seed=4, spread=20.0, scale=1e-8)


@pytest.mark.parametrize("news", [None, [3, 5, 1]])
def test_sequences_without_tokens(news):
    """Lengths of zero, and more queries than tokens: rows that see nothing."""
    lens = [0, 2, 40] if news else [0, 0, 40]
    from cublade_amd.quantization import attend_kv
    g = _gen(1)
    table, pages = _kv.make_table(lens, 16, g)
    cache = _kv.random_cache(pages, 2, 64, 16, F8, g)
    m = news or [1, 1, 1]
    q = torch.randn(sum(m), 4, 64, generator=g, device=DEV).half()
    o, lse = attend_kv(q, cache, table, _i32(lens), cu_q=_cu(news) if news else None,
                       return_lse=True)
    empty = 6 if news else 2
    assert bool((o[:empty] == 0).all()) and bool((lse[:empty] == -math.inf).all())
    assert bool((o[empty:] != 0).any()) and bool(lse[empty:].isfinite().all())
    _kv.assert_attends((o, lse), _kv.attend_ref(q, cache, table, lens, m), F16)


def test_negative_length_is_empty():
    from cublade_amd.quantization import attend_kv
    cache = _kv.random_cache(2, 1, 64, 16, I8, _gen(2))
    q = torch.ones(1, 2, 64, device=DEV).half()
    o, lse = attend_kv(q, cache, _i32([[0]]), _i32([-5]), return_lse=True)
    assert bool((o == 0).all()) and bool((lse == -math.inf).all())


@pytest.mark.parametrize("splits", [False, True])
def test_places_outside_the_pool_give_nan(splits):
    from cublade_amd.quantization import attend_kv
    g = _gen(3)
    n = 9000 if splits else 100
    lens = [n, n, n]
    table, pages = _kv.make_table(lens, 16, g)
    cache = _kv.random_cache(pages, 1, 64, 16, I8, g)
    good = table.clone()
    table[0, 3] = pages
    table[1, -1] = -1
    q = torch.randn(3, 2, 64, generator=g, device=DEV).half()
    o = attend_kv(q, cache, table, _i32(lens))
    assert bool(o[:2].isnan().all()) and bool(o[2].isfinite().all())
    o = attend_kv(q, cache, good, _i32([n, good.shape[1] * 16 + 1, 2**31 - 1]))
    assert bool(o[0].isfinite().all()) and bool(o[1:].isnan().all())
    # outside the window, an id is not looked at
    o = attend_kv(q, cache, table, _i32(lens), window=20)
    assert bool(o[0].isfinite().all()) and bool(o[1].isnan().all())


def test_empty_pool():
    from cublade_amd.quantization import QuantizedKVCache, attend_kv
    cache = QuantizedKVCache.empty(0, 1, 64, 16)
    q = torch.ones(2, 1, 64, device=DEV).half()
    o = attend_kv(q, cache, _i32([[0], [0]]), _i32([0, 3]))
    assert bool((o[0] == 0).all()) and bool(o[1].isnan().all())
    none = torch.empty(0, 1, 64, device=DEV).half()
    o, lse = attend_kv(none, cache, torch.empty(0, 1, dtype=torch.int32, device=DEV), _i32([]),
                       return_lse=True)
    assert o.shape == (0, 1, 64) and lse.shape == (0, 1)


@pytest.mark.parametrize("news", [None, [30, 30]])
def test_codes_behind_the_end_do_not_matter(news):
    """FP8 NaN codes and scales behind the sequences' ends, and in pages that
    are not theirs."""
    lens = [70, 33]
    q, cache, table, want = _check(64, 32, F8, F16, 1, 2, lens, news)
    from cublade_amd.quantization import attend_kv
    used = torch.zeros(cache.num_pages, dtype=torch.bool, device=DEV)
    nan = torch.tensor(0x7F, dtype=torch.uint8, device=DEV)
    k8, v8 = cache.k.view(torch.uint8), cache.v.view(torch.uint8)
    for b, n in enumerate(lens):
        for p in range(_kv.pages_for(n, 32)):
            pid = int(table[b, p])
            used[pid] = True
            if n - 32 * p < 32:
                k8[pid, :, n - 32 * p:] = nan
                v8[pid, :, :, n - 32 * p:] = nan
    cache.k_scale[~used] = math.nan
    cache.v_scale[~used] = math.inf
    o, lse = attend_kv(q, cache, table, _i32(lens), cu_q=_cu(news) if news else None,
                       return_lse=True)
    assert torch.equal(o, want[0]) and torch.equal(lse, want[1])


@pytest.mark.parametrize("rep,n", [(2, 40), (4, 150)])
def test_nan_reaches_only_rows_that_see_it(rep, n):
    """An FP8 NaN key makes the rows that see it NaN, a NaN value only its
    dimension of theirs; rows masked from it are as without it. A NaN query
    concerns its own row."""
    from cublade_amd.quantization import attend_kv
    q, cache, table, (base, _) = _check(64, 16, F8, BF16, 1, rep, [n], [n])
    j = n - 9
    pid, off = int(table[0, j // 16]), j % 16
    v8 = cache.v.view(torch.uint8)
    old = v8[pid, 0, 5, off].clone()
    v8[pid, 0, 5, off] = 0xFF
    o = attend_kv(q, cache, table, _i32([n]), cu_q=_cu([n]))
    assert torch.equal(o[:j], base[:j]) and bool(o[j:, :, 5].isnan().all())
    rest = [i for i in range(64) if i != 5]
    assert torch.equal(o[j:][..., rest], base[j:][..., rest])
    v8[pid, 0, 5, off] = old
    cache.k.view(torch.uint8)[pid, 0, off, 7] = 0x7F
    o = attend_kv(q, cache, table, _i32([n]), cu_q=_cu([n]))
    assert torch.equal(o[:j], base[:j]) and bool(o[j:].isnan().all())
    cache.k.view(torch.uint8)[pid, 0, off, 7] = 0
    q2 = q.clone()
    base = attend_kv(q, cache, table, _i32([n]), cu_q=_cu([n]))
    q2[3, 0, 2] = math.nan
    o = attend_kv(q2, cache, table, _i32([n]), cu_q=_cu([n]))
    assert bool(o[3, 0].isnan().all())
    o[3, 0] = base[3, 0]
    assert torch.equal(o, base)


def test_page_scales_that_are_no_numbers():
    """A poisoned page (an infinite scale) concerns the rows that see a token of
    it; a zero scale stands for zeros."""
    from cublade_amd.quantization import attend_kv
    n = 100
    q, cache, table, (base, _) = _check(64, 16, I8, F16, 1, 2, [n], [n])
    for scale in (cache.k_scale, cache.v_scale):
        pid = int(table[0, 4])
        old = scale[pid].clone()
        cache.k[pid] = 0
        clean = attend_kv(q, cache, table, _i32([n]), cu_q=_cu([n]))
        scale[pid] = math.inf
        o = attend_kv(q, cache, table, _i32([n]), cu_q=_cu([n]))
        assert torch.equal(o[:64], base[:64]) and bool(o[64:].isnan().all())
        scale[pid] = 0
        got = attend_kv(q, cache, table, _i32([n]), cu_q=_cu([n]), return_lse=True)
        _kv.assert_attends(got, _kv.attend_ref(q, cache, table, [n], [n]), F16)
        scale[pid] = old
        assert torch.equal(clean, attend_kv(q, cache, table, _i32([n]), cu_q=_cu([n])))


def test_strided_and_misaligned_queries():
    from cublade_amd.quantization import attend_kv
    g, lens = _gen(4), [40, 90]
    table, pages = _kv.make_table(lens, 16, g)
    cache = _kv.random_cache(pages, 2, 64, 16, I8, g)
    wide = torch.randn(2, 12, 72, generator=g, device=DEV).half()
    for q in (wide[:, 2:6, :64], wide[:, 2:6, 3:67], wide[:, ::3, 8:], wide.transpose(0, 1)[:2][..., :64].repeat(1, 2, 1)):
        assert torch.equal(attend_kv(q, cache, table, _i32(lens)),
                           attend_kv(q.contiguous(), cache, table, _i32(lens)))
    t2 = torch.stack([table, table], -1)[..., 1]
    assert torch.equal(attend_kv(wide[:, :4, :64], cache, t2, _i32(lens)),
                       attend_kv(wide[:, :4, :64], cache, table, _i32(lens)))
    one = table[:1].expand(2, -1)
    o = attend_kv(wide[:, :4, :64], cache, one, _i32([40, 40]))
    assert torch.equal(o[1:], attend_kv(wide[1:, :4, :64], cache, table[:1], _i32([40])))


def test_large_queries():
    """bf16 queries beyond fp16's range, and tiny ones."""
    from cublade_amd.quantization import attend_kv
    g, lens = _gen(5), [100]
    table, pages = _kv.make_table(lens, 16, g)
    cache = _kv.random_cache(pages, 1, 64, 16, I8, g)
    for mul, scale in ((1e30, 1e-31), (1e-30, 1e29), (0.0, 1.0)):
        q = (torch.randn(1, 4, 64, generator=g, device=DEV) * mul).bfloat16()
        got = attend_kv(q, cache, table, _i32(lens), scale=scale, return_lse=True)
        ref = _kv.attend_ref(q, cache, table, lens, [1], scale=scale)
        _kv.assert_attends(got, ref, BF16, mul)


def test_runs_are_equal_and_streams_independent():
    """The same bits every time, also on another stream and replayed from a
    graph, and for a call whose workspace has no room for splits."""
    from cublade_amd.quantization import append_kv, attend_kv
    g, lens = _gen(6), [5000, 77]
    table, pages = _kv.make_table(lens, 64, g)
    cache = _kv.random_cache(pages, 2, 128, 64, I8, g)
    q = torch.randn(2, 8, 128, generator=g, device=DEV).bfloat16()
    n = _i32(lens)
    want = attend_kv(q, cache, table, n)
    for _ in range(3):
        assert torch.equal(attend_kv(q, cache, table, n), want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    k = torch.randn(2, 2, 128, generator=g, device=DEV).bfloat16()
    rope = _kv.tables(6000, 128)
    saved = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        assert torch.equal(attend_kv(q, cache, table, n), want)
        qr = append_kv(cache, k, k, table, n, rope=rope, q=q)
        after = attend_kv(qr, cache, table, n)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            gq = append_kv(cache, k, k, table, n, rope=rope, q=q)
            go = attend_kv(gq, cache, table, n)
        for _ in range(3):
            for t, o in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), saved):
                t.copy_(o)
            go.zero_()
            graph.replay()
            s.synchronize()
            assert torch.equal(gq, qr) and torch.equal(go, after)
            assert torch.equal(attend_kv(qr, cache, table, n), after)


def test_small_workspace_gives_the_same_within_rounding():
    import ctypes
    from cublade_amd import _abi
    from cublade_amd.bindings.hip import kv_cache as kvb
    g, lens = _gen(7), [6000]
    table, pages = _kv.make_table(lens, 64, g)
    cache = _kv.random_cache(pages, 1, 64, 64, I8, g)
    q = torch.randn(1, 4, 64, generator=g, device=DEV).half()
    ref = _kv.attend_ref(q, cache, table, lens, [1])
    L, by = _abi.lib(), ctypes.byref
    batch, keep = kvb._batch(cache.device, 1, table, _i32(lens), None)
    heads, _ = kvb._heads(q, cache.device, None, None, 64, None, "q")
    full = L.cbq_kv_attend_ws_bytes(by(cache._view), by(batch), 4, 0)
    assert full > _abi.WS_CTRL_BYTES
    for nbytes in (full, full // 3, _abi.WS_CTRL_BYTES, 0):
        ws = torch.zeros(max(nbytes, 256), dtype=torch.uint8, device=DEV)
        o = torch.empty_like(q)
        lse = torch.empty(1, 4, device=DEV)
        _abi.check(L.cbq_kv_attend(by(cache._view), by(batch), _abi.F16, by(heads), 4, 0.125, 1, 0, 0,
                                   ws.data_ptr() if nbytes else None, nbytes, o.data_ptr(),
                                   lse.data_ptr(), _abi.stream_handle(cache.device)), "attend")
        _kv.assert_attends((o, lse), ref, F16, nbytes)
        torch.cuda.synchronize()


@pytest.mark.parametrize("store,dt", [(I8, BF16), (F8, F16), (F8, BF16)])
@pytest.mark.parametrize("d,page", [(80, 16), (96, 32), (96, 256)])
def test_prompts_of_96_wide_tiles(d, page, store, dt):
    """Head sizes over 64 and up to 96 with many rows: the tiles are 96 wide, and
    lanes of a workgroup's second piece have none."""
    _check(d, page, store, dt, 2, 4, [1, 130, 64, 333, 129], [1, 130, 0, 200, 33])
    _check(d, page, store, dt, 1, 2, [500], [300], window=70)
    _check(d, page, store, dt, 2, 2, [200, 90], [200, 70], causal=False)


@pytest.mark.parametrize("d", [80, 96])
@pytest.mark.parametrize("dim", [3, 63, 64, 79])
def test_nan_value_in_96_wide_tiles(d, dim):
    """One FP8 NaN value reaches its dimension of the rows that see its token, in
    either piece of a thread's dimensions."""
    from cublade_amd.quantization import attend_kv
    n, rep = 150, 4
    q, cache, table, (base, _) = _check(d, 32, F8, BF16, 1, rep, [n], [n])
    j = 101
    cache.v.view(torch.uint8)[int(table[0, j // 32]), 0, dim, j % 32] = 0x7F
    o = attend_kv(q, cache, table, _i32([n]), cu_q=_cu([n]))
    rest = [i for i in range(d) if i != dim]
    assert bool(o[j:, :, dim].isnan().all())
    assert torch.equal(o[:j], base[:j]) and torch.equal(o[j:][..., rest], base[j:][..., rest])


@pytest.mark.parametrize("store,dt", [(I8, BF16), (F8, F16)])
@pytest.mark.parametrize("d,page", [(128, 64), (80, 16), (64, 32), (192, 16), (256, 128)])
@pytest.mark.parametrize("window", [1, 70, 1024])
def test_window_over_prompts_and_single_tokens(d, page, store, dt, window):
    """Single tokens, drafted ones and prompts under a window that one launch takes
    them all with: sequences that bring nothing, hold nothing, or bring more than
    they hold."""
    _check(d, page, store, dt, 2, 4, [1300, 900, 1, 0, 40, 65, 700, 3], [150, 1, 1, 0, 9, 1, 33, 1],
           window=window)
    _check(d, page, store, dt, 1, 4, [5, 200, 0, 400], [9, 150, 2, 1], window=window)


@pytest.mark.parametrize("store,dt", [(I8, BF16), (F8, F16)])
def test_window_in_two_launches(store, dt):
    """Windows and batches past what one launch takes."""
    _check(64, 32, store, dt, 2, 4, [2500, 1900, 70, 2100], [150, 1, 1, 5], window=1500)
    n = 170
    _check(64, 16, store, dt, 2, 32, [100 + i for i in range(n)],
           [64 if i % 40 == 0 else 1 for i in range(n)], window=50)


def test_window_of_one_launch_keeps_nan_to_its_rows():
    """An FP8 NaN value ahead of a window, or outside another sequence, reaches
    no row; inside, its dimension of the rows that see it."""
    from cublade_amd.quantization import attend_kv
    lens, news = [300, 200, 90], [100, 1, 1]
    q, cache, table, (base, _) = _check(96, 32, F8, F16, 1, 4, lens, news, window=40)
    args = (table, _i32(lens))
    v8 = cache.v.view(torch.uint8)
    v8[int(table[1, 4]), 0, 7, 130 % 32] = 0x7F      # token 130 of 200: before its window
    o = attend_kv(q, cache, *args, cu_q=_cu(news), window=40)
    assert torch.equal(o, base)
    v8[int(table[1, 5]), 0, 7, 170 % 32] = 0x7F      # token 170: inside
    o = attend_kv(q, cache, *args, cu_q=_cu(news), window=40)
    assert bool(o[100, :, 7].isnan().all())
    rest = [i for i in range(96) if i != 7]
    assert torch.equal(o[100][:, rest], base[100][:, rest])
    assert torch.equal(o[:100], base[:100]) and torch.equal(o[101:], base[101:])


@pytest.mark.parametrize("news", [None, [40, 40, 40, 40]])
@pytest.mark.parametrize("n", [40, 9000])
def test_lse_is_nan_where_every_score_is(n, news):
    """-infinity is the log-sum-exp of rows that see no key, not of rows that
    see none but NaN scores: queries of NaN, pages that are not in the pool."""
    from cublade_amd.quantization import attend_kv
    g = _gen(21)
    lens = [n, n, n, 0]
    table, pages = _kv.make_table(lens, 16, g)
    cache = _kv.random_cache(pages, 1, 64, 16, I8, g)
    table[1] = -1
    t = 4 if news is None else sum(news)
    q = torch.randn(t, 2, 64, generator=g, device=DEV).half()
    per = t // 4
    q[:per, 0] = math.nan
    o, lse = attend_kv(q, cache, table, _i32(lens), cu_q=None if news is None else _cu(news),
                       return_lse=True)
    for x in (o, lse):
        assert bool(x[:per, 0].isnan().all()) and bool(x[:per, 1].isfinite().all())
        assert bool(x[per:2 * per].isnan().all()) and bool(x[2 * per:3 * per].isfinite().all())
    assert bool((o[3 * per:] == 0).all()) and bool((lse[3 * per:] == -math.inf).all())


@pytest.mark.parametrize("news", [None, [70]])
def test_largest_finite_queries(news):
    """bf16 queries of the last binade, [2^127, 2^128), whose scores are finite."""
    from cublade_amd.quantization import attend_kv
    g, lens = _gen(23), [100]
    table, pages = _kv.make_table(lens, 16, g)
    cache = _kv.random_cache(pages, 1, 64, 16, I8, g)
    t, scale = 1 if news is None else 70, 2.0 ** -124
    q = (torch.rand(t, 4, 64, generator=g, device=DEV) * 2 - 1) * 2.0 ** 127
    q[:, :, 5] = 2.0 ** 127 * 1.5
    q = q.bfloat16()
    got = attend_kv(q, cache, table, _i32(lens), scale=scale, return_lse=True,
                    cu_q=None if news is None else _cu(news))
    assert bool(got[0].isfinite().all())
    ref = _kv.attend_ref(q, cache, table, lens, news or [1], scale=scale)
    _kv.assert_attends(got, ref, BF16, news)
