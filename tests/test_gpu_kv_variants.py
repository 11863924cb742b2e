"""Forms of the cache's kernels that sizes choose: 256-row tiles of prompts, the
single-token append of wide heads, one wave per token of queries; and attention
over long contexts within a bound that a lost block of values exceeds."""
from __future__ import annotations

import pytest
import torch

from tests import _kv, _kv_tight

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


def _check(d, page, store, dt, hkv, rep, lens, news=None, seed=0, spread=1.0, width=None, **kw):
    from cublade_amd.quantization import attend_kv
    g = _gen(seed)
    m = news or [1] * len(lens)
    table, pages = _kv.make_table(lens, page, g, width)
    cache = _kv.random_cache(pages, hkv, d, page, store, g, spread)
    q = torch.randn(sum(m), hkv * rep, d, generator=g, device=DEV).to(dt)
    extra = {k: kw.pop(k) for k in ("max_length",) if k in kw}
    got = attend_kv(q, cache, table, _i32(lens), cu_q=_cu(news) if news else None, return_lse=True,
                    **kw, **extra)
    ref = _kv_tight.attend_tight(q, cache, table, lens, m, **kw)
    over = _kv_tight.excess(got, ref, dt)
    assert over <= 1, over
    return q, cache, table, got


# Long contexts, their keys cut into ranges or not, and prompts -----------------
@pytest.mark.parametrize("store", [I8, F8])
@pytest.mark.parametrize("kw", [{}, {"max_length": 9000}, {"width": 2000}, {"window": 3000}])
def test_single_tokens_over_long_contexts(store, kw):
    _check(128, 64, store, BF16, 2, 4, [9000, 3, 700], **kw)
    _check(64, 16, store, F16, 1, 8, [20001, 64], **kw)


@pytest.mark.parametrize("store", [I8, F8])
def test_several_tokens_over_long_contexts(store):
    _check(64, 16, store, F16, 1, 8, [20001], [5])
    _check(64, 16, store, F16, 1, 8, [20001], [5], window=3000)
    _check(128, 64, store, BF16, 2, 4, [4100], [600])
    _check(96, 32, store, F16, 2, 2, [5000, 900, 77], [70, 900, 1])
    _check(256, 128, store, F16, 1, 2, [3000], [65])


@pytest.mark.parametrize("store", [I8, F8])
@pytest.mark.parametrize("news", [None, [40, 100]])
def test_scales_far_apart(store, news):
    _check(64, 16, store, F16, 2, 2, [400, 100], news, seed=3, spread=20.0, scale=1e-8)


# 256-row tiles ---------------------------------------------------------------
def _full_tiles(hkv, rep, off=0):
    """Tokens of one sequence whose rows, in tiles of 256, make one for each CU:
    the form with 8 waves takes these (head sizes 97 to 128)."""
    cus = torch.cuda.get_device_properties(DEV).multi_processor_count
    return 256 * (cus // hkv) // rep - off


@pytest.mark.parametrize("store,dt", [(I8, BF16), (F8, F16)])
@pytest.mark.parametrize("d,page", [(128, 64), (112, 16)])
def test_prompt_in_tiles_of_256(d, page, store, dt):
    n = _full_tiles(8, 4)
    _check(d, page, store, dt, 8, 4, [n], [n])
    # rows that are no multiple of a tile's, over earlier tokens
    n = _full_tiles(8, 4, off=7)
    _check(d, page, store, dt, 8, 4, [n + 333], [n])


@pytest.mark.parametrize("store,dt", [(I8, F16), (F8, BF16)])
def test_tiles_of_256_under_masks(store, dt):
    n = _full_tiles(16, 4)
    _check(128, 32, store, dt, 16, 4, [n + 50], [n], window=300)
    _check(128, 32, store, dt, 16, 4, [n], [n], causal=False)
    _check(128, 32, store, dt, 16, 4, [n - 20], [n])        # more queries than tokens


@pytest.mark.parametrize("store,dt", [(I8, BF16), (F8, F16)])
def test_tiles_of_256_of_several_sequences(store, dt):
    cus = torch.cuda.get_device_properties(DEV).multi_processor_count
    # 3 tiles for each CU in all: 16 kv heads, 8 query heads each
    n = 3 * cus * 256 // (16 * 8) // 4 + 40
    _check(128, 64, store, dt, 16, 8, [n, n + 100, 5, n, n + 1], [n - 5, n, 5, n - 1, n])


@pytest.mark.parametrize("dim", [0, 63, 64, 127])
def test_nan_value_in_tiles_of_256(dim):
    """An FP8 NaN value, near each end of a wave's share of the dimensions, in
    keys that only some rows of a tile see: its dimension of the rows that do."""
    from cublade_amd.quantization import attend_kv
    n = _full_tiles(16, 4)
    q, cache, table, (base, _) = _check(128, 32, F8, BF16, 16, 4, [n], [n], seed=dim)
    j, h = n - 37 - dim, 5
    cache.v.view(torch.uint8)[int(table[0, j // 32]), h, dim, j % 32] = 0xFF
    o = attend_kv(q, cache, table, _i32([n]), cu_q=_cu([n]))
    heads = slice(4 * h, 4 * h + 4)
    assert bool(o[j:, heads, dim].isnan().all())
    o[j:, heads, dim] = base[j:, heads, dim]
    assert torch.equal(o, base)


# Append ----------------------------------------------------------------------
def _append(d, rot, inter, page, store, dt, hkv, rep, lens, news, seed):
    from cublade_amd.quantization import append_kv
    g = _gen(seed)
    m = news or [1] * len(lens)
    table, pages = _kv.make_table(lens, page, g)
    cache = _kv.random_cache(pages, hkv, d, page, store, g)
    model = _kv.CacheModel(cache)
    t = sum(m)
    # heads of a token differ by powers of two: some pages grow, others keep their scale
    qkv = torch.randn(t, hkv * (rep + 2), d, generator=g, device=DEV)
    qkv *= torch.exp2(torch.randint(-3, 5, (t, hkv * (rep + 2), 1), generator=g, device=DEV).float())
    qkv = qkv.to(dt)
    q, k, v = qkv[:, :hkv * rep], qkv[:, hkv * rep:hkv * (rep + 1)], qkv[:, hkv * (rep + 1):]
    pos = torch.cat([torch.arange(n - c, n) for n, c in zip(lens, m)]).to(DEV)
    rope = _kv.tables(max(lens), rot) if rot else None
    out = append_kv(cache, k, v, table, _i32(lens), cu_new=_cu(news) if news else None, rope=rope,
                    interleaved=inter, q=q)
    rk, rq = (_kv.rotate_f32(x, pos, *rope, inter) if rot else x.float() for x in (k, q))
    model.append(rk, v, table, lens, m)
    model.assert_equal(cache)
    assert torch.equal(out, rq.to(dt))


@pytest.mark.parametrize("store,dt", [(I8, BF16), (F8, F16)])
@pytest.mark.parametrize("d,rot,inter", [(144, 144, False), (192, 96, True), (256, 256, False),
                                         (256, 40, False), (176, 0, False)])
@pytest.mark.parametrize("hkv", [1, 2, 3])
def test_single_tokens_of_wide_heads(d, rot, inter, store, dt, hkv):
    """Heads over 128 wide, two to a wave, an odd number of them, in pages that
    begin, are begun and grow."""
    _append(d, rot, inter, 32, store, dt, hkv, 2, [1, 2, 32, 33, 47, 64, 65, 200], None, d + hkv)


@pytest.mark.parametrize("rot,inter", [(0, False), (64, False), (32, False), (64, True), (20, False)])
@pytest.mark.parametrize("step", [True, False])
def test_queries_of_more_than_1024_tokens(rot, inter, step):
    if step:
        lens, news = [1 + (5 * i) % 40 for i in range(1100)], None
    else:
        lens, news = [700, 900, 30], [600, 500, 0]
    _append(64, rot, inter, 16, I8, BF16, 1, 9, lens, news, rot + step)
