"""append_kv and dequantize_kv on the GPU: codes and scales equal to the
formulas in fp32 (the order of roundings is part of the definition), values
within the quantisation's bounds of the rotated inputs in 64 bits, and what is
dropped or poisoned rather than read or written out of range."""
from __future__ import annotations

import math

import pytest
import torch

from tests import _kv

pytestmark = pytest.mark.gpu
DEV = "cuda"
I8, F8 = torch.int8, torch.float8_e4m3fn


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _cu(news):
    c = [0]
    for n in news:
        c.append(c[-1] + n)
    return torch.tensor(c, dtype=torch.int32, device=DEV)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


CASES = [
    # d, rot, interleaved, page, store, dtype, hkv, rep, lens, news
    (128, 128, False, 64, I8, torch.bfloat16, 8, 4, [1, 2, 64, 65, 700], None),
    (64, 64, True, 16, F8, torch.float16, 2, 1, [1, 16, 17, 33, 48], None),
    (16, 16, False, 16, I8, torch.float16, 1, 3, [40], [40]),
    (256, 128, False, 256, F8, torch.bfloat16, 2, 2, [256, 700, 5], [256, 300, 5]),
    (80, 80, False, 32, I8, torch.bfloat16, 3, 2, [31, 32, 33, 100, 64, 90], [31, 1, 33, 0, 40, 3]),
    (96, 36, False, 32, F8, torch.float16, 2, 3, [70, 1, 129], [70, 1, 64]),
    (112, 10, True, 128, I8, torch.float16, 2, 1, [300, 128], [200, 128]),
    (192, 0, False, 64, F8, torch.bfloat16, 1, 8, [64, 65], [1, 65]),
    # more sequences than lanes of a wave, most of them bringing nothing
    (32, 32, False, 16, I8, torch.bfloat16, 1, 2, [(7 * i) % 50 + 2 for i in range(150)],
     [2 if i % 3 == 0 else 0 for i in range(150)]),
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_append_matches_the_formulas(case):
    from cublade_amd.quantization import append_kv, dequantize_kv
    d, rot, inter, page, store, dt, hkv, rep, lens, news = CASES[case]
    g = _gen(case)
    step = news is None
    news = [1] * len(lens) if step else news
    table, pages = _kv.make_table(lens, page, g)
    cache = _kv.random_cache(pages, hkv, d, page, store, g)
    model = _kv.CacheModel(cache)
    t = sum(news)
    # values that make begun pages keep their scale, and some that make it grow
    qkv = torch.randn(t, hkv * (rep + 2), d, generator=g, device=DEV)
    qkv *= torch.exp2(torch.randint(-2, 5, (t, 1, 1), generator=g, device=DEV).float())
    qkv = qkv.to(dt)
    q, k, v = qkv[:, :hkv * rep], qkv[:, hkv * rep:hkv * (rep + 1)], qkv[:, hkv * (rep + 1):]
    cos, sin = _kv.tables(max(lens), rot) if rot else (None, None)
    pos = torch.cat([torch.arange(n - m, n) for n, m in zip(lens, news)]).to(DEV)
    out = append_kv(cache, k, v, table, _i32(lens), cu_new=None if step else _cu(news),
                    rope=(cos, sin) if rot else None, interleaved=inter, q=q)
    rk = _kv.rotate_f32(k, pos, cos, sin, inter) if rot else k.float()
    rq = _kv.rotate_f32(q, pos, cos, sin, inter) if rot else q.float()
    model.append(rk, v, table, lens, news)
    model.assert_equal(cache, CASES[case])
    assert bool((out == rq.to(dt)).all())

    # the values in 64 bits: half a step of the codes for the new tokens
    rk64 = _kv.rotate_ref(k, pos, cos, sin, inter) if rot else k.double()
    at = 0
    for b, (n, m) in enumerate(zip(lens, news)):
        if m:
            kk, vv = _kv.values(cache, table, b, n)
            ids = table[b, :_kv.pages_for(n, page)].long()
            for got, want, scale in ((kk, rk64, cache.k_scale), (vv, v.double(), cache.v_scale)):
                want = want[at:at + m].transpose(0, 1)
                s = scale[ids].double().repeat_interleave(page, 0)[n - m:n].t()[:, :, None]
                err = (got[:, n - m:] - want).abs()
                half = 0.5 * s if store == I8 else torch.maximum(want.abs() * 2.0 ** -4, s * 2.0 ** -10)
                # the rotation and the product with 1 / scale are rounded to 32 bits
                assert bool((err <= half + 127 * s * 2.0 ** -21 + want.abs() * 2.0 ** -21).all())
        at += m
    kd, vd = dequantize_kv(cache, table[table >= 0].to(torch.int32), dt)
    ids = table[table >= 0].long()
    assert bool((kd == (cache.k[ids].float() * cache.k_scale[ids][:, :, None, None]).to(dt)).all())
    want = (cache.v[ids].float() * cache.v_scale[ids][:, :, None, None]).transpose(2, 3).to(dt)
    assert bool((vd == want).all())


@pytest.mark.parametrize("store", [I8, F8])
def test_token_by_token_stays_within_a_step(store):
    """A page filled one token at a time, each larger than the ones before: the
    scale grows often, and every value stays within one step (INT8) of the
    final scale, or 2^-3 of itself (FP8, two roundings), of what was given."""
    from cublade_amd.quantization import QuantizedKVCache, append_kv
    g, page, d = _gen(5), 64, 64
    cache = QuantizedKVCache.empty(3, 2, d, page, store)
    x = torch.randn(page, 2, d, generator=g, device=DEV)
    x = (x * torch.logspace(-3, 2, page, device=DEV)[:, None, None]).to(torch.bfloat16)
    y = x.flip(2).contiguous()
    table = _i32([[1]])
    for t in range(page):
        append_kv(cache, x[t:t + 1], y[t:t + 1], table, _i32([t + 1]))
    for got, want, s in zip(_kv.values(cache, table, 0, page), (x, y),
                            (cache.k_scale[1], cache.v_scale[1])):
        want = want.double().transpose(0, 1)
        err, s = (got - want).abs(), s.double()[:, None, None]
        q = _kv.QMAX[store]
        assert bool((want.abs().amax((1, 2)) <= q * s.flatten() * (1 + 2.0 ** -20)).all())
        assert bool((want.abs().amax((1, 2)) > q * s.flatten() * 0.49).all())
        limit = s if store == I8 else torch.maximum(want.abs() / 8, s * 2.0 ** -9)
        assert bool((err <= limit * (1 + 2.0 ** -18)).all())


def test_strides_and_alignment():
    """Heads first, misaligned and non-contiguous inputs, an expanded page
    table and int32 views give what contiguous ones do."""
    from cublade_amd.quantization import append_kv
    g, lens, page, d, hkv = _gen(6), [20, 40], 16, 48, 2
    table, pages = _kv.make_table(lens, page, g)
    base = torch.randn(hkv, 60, d + 8, generator=g, device=DEV).half()
    k0 = base[:, :, :d].transpose(0, 1)
    v0 = base[:, :, 4:d + 4].transpose(0, 1)      # 8-byte aligned rows
    q0 = torch.randn(60, d, 4, generator=g, device=DEV).half().transpose(1, 2)
    rope = _kv.tables(64, 32)
    rope_off = tuple(torch.cat([torch.zeros(1, device=DEV), r.flatten()])[1:].view_as(r) for r in rope)
    res = []
    for mk in (lambda t: t.contiguous(), lambda t: t):
        cache = _kv.random_cache(pages, hkv, d, page, I8, _gen(1))
        wide = torch.stack([table, table], -1)[..., 0] if res else table
        out = append_kv(cache, mk(k0), mk(v0), wide, _i32(lens), cu_new=_cu(lens),
                        rope=rope_off if res else rope, q=mk(q0))
        res.append((out, cache))
    (a, ca), (b, cb) = res
    assert torch.equal(a, b) and torch.equal(ca.k, cb.k) and torch.equal(ca.v, cb.v)
    assert torch.equal(ca.k_scale, cb.k_scale) and torch.equal(ca.v_scale, cb.v_scale)


def test_positions_and_rows_outside_the_tables():
    from cublade_amd.quantization import append_kv, dequantize_kv
    g, page, d = _gen(7), 16, 32
    cache = _kv.random_cache(4, 1, d, page, I8, g)
    cos, sin = _kv.tables(50, d)
    table, lens, news = _i32([[0], [1], [2]]), [3, 2, 5], [3, 2, 5]
    x = torch.randn(10, 1, d, generator=g, device=DEV).half()
    pos = torch.tensor([9, 7, 0, 49, 1, 3, 3, 50, 2, 2], device=DEV)     # token 7 has no row
    model = _kv.CacheModel(cache)
    out = append_kv(cache, x, x, table, _i32(lens), cu_new=_cu(news), rope=(cos, sin),
                    positions=pos, q=x)
    ok = pos.clamp(max=49)
    model.append(_kv.rotate_f32(x, ok, cos, sin, False), x, table, lens, news)
    assert torch.equal(model.ks[:2], cache.k_scale[:2]) and torch.equal(model.k[:2], cache.k[:2])
    assert torch.equal(model.vs, cache.v_scale)
    want = _kv.rotate_f32(x, ok, cos, sin, False).half()
    keep = torch.arange(10, device=DEV) != 7
    assert torch.equal(out[keep], want[keep]) and bool(out[7].isnan().all())
    assert math.isinf(float(cache.k_scale[2]))
    assert bool(dequantize_kv(cache, _i32([2]))[0][0, 0, :5].isnan().all())


def test_out_of_range_places_are_dropped():
    """Page ids outside the pool, pages past the table's width, more new tokens
    than the length has: those tokens are not stored, the others are."""
    from cublade_amd.quantization import append_kv, attend_kv, dequantize_kv
    g, page, d = _gen(8), 16, 32
    cache = _kv.random_cache(4, 1, d, page, I8, g)
    before = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    table = _i32([[0, 4], [-1, 1], [2, 3]])
    lens, news = [32, 32, 40], [32, 32, 40]
    x = torch.randn(104, 1, d, generator=g, device=DEV).half()
    append_kv(cache, x, x, table, _i32(lens), cu_new=_cu(news))
    model = _kv.CacheModel(type(cache)(*before))
    big = [0, 1, 2, 3]
    for pid, at in zip(big, (0, 48, 64, 80)):
        xs = x[at:at + 16].float()
        model.put(xs, model.k, model.ks, [pid], 0)
        model.put(xs, model.v, model.vs, [pid], 0)
    model.assert_equal(cache)
    k, v = dequantize_kv(cache, _i32([0, 4, -1, 3]), torch.float16)
    assert bool(k[1:3].isnan().all() and v[1:3].isnan().all() and k[[0, 3]].isfinite().all())
    o = attend_kv(x[[0, 1, 2]], cache, table, _i32(lens))
    assert bool(o.isnan().all())
    # a length below the number of new tokens: the first ones have no place
    keep = cache.k.clone()
    append_kv(cache, x[:5], x[:5], _i32([[3]]), _i32([2]), cu_new=_cu([5]))
    model.put(x[3:5].float(), model.k, model.ks, [3], 0)
    model.put(x[3:5].float(), model.v, model.vs, [3], 0)
    model.assert_equal(cache)
    assert torch.equal(keep[:3], cache.k[:3])
    # lengths of zero and below: nothing at all
    append_kv(cache, x[:2], x[:2], _i32([[3], [2]]), _i32([0, -4]))
    model.assert_equal(cache)


@pytest.mark.parametrize("store", [I8, F8])
def test_values_that_are_no_numbers(store):
    """Zeros, NaN and infinities: zeros give the smallest scale; NaN is left out
    of the maximum and becomes code 0 (INT8) or NaN (FP8), as in
    quantize_tensor; an infinity makes its page's scale infinite."""
    from cublade_amd.quantization import QuantizedKVCache, append_kv, dequantize_kv
    cache = QuantizedKVCache.empty(3, 1, 16, 16, store)
    k = torch.ones(4, 1, 16, device=DEV).half()
    v = torch.zeros_like(k)
    k[1, 0, 3] = math.nan
    append_kv(cache, k, v, _i32([[0]]), _i32([4]), cu_new=_cu([4]))
    q = _kv.QMAX[store]
    assert abs(float(cache.k_scale[0]) * q - 1) < 1e-6
    assert abs(float(cache.v_scale[0]) / (1e-12 / q) - 1) < 1e-6
    kd, vd = dequantize_kv(cache, _i32([0]), torch.float16)
    assert bool((vd == 0).all())
    bad = kd[0, 0, 1, 3]
    assert bool(bad.isnan()) if store == F8 else float(bad) == 0
    # the zeros' page then gets ones, then an infinity
    append_kv(cache, k[:1], k[:1], _i32([[0]]), _i32([5]))
    vd = dequantize_kv(cache, _i32([0]), torch.float16)[1]
    assert bool((vd[0, 0, :4] == 0).all())
    assert bool(((vd[0, 0, 4] - 1).abs() <= (2.0 ** -4 if store == F8 else 1 / 127)).all())
    k[0, 0, 0] = math.inf
    append_kv(cache, k[:1], k[:1], _i32([[0]]), _i32([6]))
    assert math.isinf(float(cache.k_scale[0]))
    assert bool(dequantize_kv(cache, _i32([0]), torch.float16)[0].isnan().all())
    assert float(cache.k_scale[1]) == 0


def test_scale_zero_stands_for_zeros():
    """A begun page whose scale is 0 (a zero-filled pool): its codes stand for
    zeros, and stay zeros when the page gets its first values."""
    from cublade_amd.quantization import append_kv, dequantize_kv
    g = _gen(9)
    cache = _kv.random_cache(2, 1, 16, 16, I8, g)
    cache.k_scale.zero_()
    cache.v_scale.zero_()
    x = torch.randn(1, 1, 16, generator=g, device=DEV).half()
    append_kv(cache, x, x, _i32([[1]]), _i32([6]))
    for t in dequantize_kv(cache, _i32([1]), torch.float16):
        assert bool((t[0, 0, :5] == 0).all())
        limit = float(x.abs().max()) * (1 / 254 + 2.0 ** -11)
        assert bool(((t[0, 0, 5].double() - x[0, 0].double()).abs() <= limit).all())


def test_empty_calls():
    from cublade_amd.quantization import QuantizedKVCache, append_kv, dequantize_kv
    cache = QuantizedKVCache.empty(0, 2, 32, 16)
    none = torch.empty(0, 2, 32, device=DEV).half()
    table, lens = torch.empty(0, 4, dtype=torch.int32, device=DEV), _i32([])
    assert append_kv(cache, none, none, table, lens) is None
    assert append_kv(cache, none, none, table, lens, q=none).shape == (0, 2, 32)
    k, v = dequantize_kv(cache, _i32([]))
    assert k.shape == v.shape == (0, 2, 16, 32)


def test_offsets_past_32_bits():
    """A pool of more than 2^32 bytes on either side, its last page used."""
    from cublade_amd.quantization import QuantizedKVCache, append_kv, attend_kv, dequantize_kv
    pages, hkv, d, page = (1 << 32) // (8 * 128 * 128) + 2, 8, 128, 128
    cache = QuantizedKVCache.empty(pages, hkv, d, page)
    assert cache.k.numel() > 1 << 32
    x = torch.randn(page, hkv, d, generator=_gen(10), device=DEV).half()
    last = _i32([[pages - 1]])
    append_kv(cache, x, x, last, _i32([page]), cu_new=_cu([page]))
    k, v = dequantize_kv(cache, last[0], torch.float16)
    # half a step of the codes, and one rounding to fp16
    limit = float(x.abs().max()) * (1 / 254 + 2.0 ** -11)
    assert float((k[0].double() - x.double().transpose(0, 1)).abs().max()) <= limit
    assert float((v[0].double() - x.double().transpose(0, 1)).abs().max()) <= limit
    assert int((cache.k[0] != 0).sum()) == 0 and int((cache.v[0] != 0).sum()) == 0
    o, lse = attend_kv(x[:1], cache, last, _i32([page]), return_lse=True)
    _kv.assert_attends((o, lse), _kv.attend_ref(x[:1], cache, last, [page], [1]), torch.float16)


@pytest.mark.parametrize("store", [I8, F8])
@pytest.mark.parametrize("begun", [0, 3, 6])
def test_rotation_table_ends_inside_a_page(store, begun):
    """Half of each head rotated, tokens past the table in the second page only:
    the first page, begun or not, is as without them; their page's keys are lost,
    its values and all other queries are not."""
    from cublade_amd.quantization import append_kv
    g, page, d, rot, n = _gen(11), 32, 64, 32, 45
    cache = _kv.random_cache(3, 2, d, page, store, g)
    model = _kv.CacheModel(cache)
    cos, sin = _kv.tables(37, rot)
    table, new = _i32([[2, 0]]), n - begun
    k = torch.randn(new, 2, d, generator=g, device=DEV).bfloat16()
    v = torch.randn(new, 2, d, generator=g, device=DEV).bfloat16()
    q = torch.randn(new, 4, d, generator=g, device=DEV).bfloat16()
    out = append_kv(cache, k, v, table, _i32([n]), cu_new=_cu([new]), rope=(cos, sin), q=q)
    pos = torch.arange(begun, n, device=DEV)
    ok = pos.clamp(max=36)
    model.append(_kv.rotate_f32(k, ok, cos, sin, False), v, table, [n], [new])
    keep = [1, 2]
    assert torch.equal(cache.k_scale[keep], model.ks[keep])
    assert torch.equal(cache.k.view(torch.uint8)[keep], model.k.view(torch.uint8)[keep])
    assert torch.equal(cache.v_scale, model.vs)
    assert torch.equal(cache.v.view(torch.uint8).transpose(2, 3), model.v.view(torch.uint8))
    assert bool(cache.k_scale[0].isinf().all())
    want = _kv.rotate_f32(q, ok, cos, sin, False).bfloat16()
    here = pos < 37
    assert torch.equal(out[here], want[here])
    assert bool(out[~here][..., :rot].isnan().all())
    assert torch.equal(out[~here][..., rot:], q[~here][..., rot:])


@pytest.mark.parametrize("store", [I8, F8])
@pytest.mark.parametrize("chunk", [False, True])
@pytest.mark.parametrize("big", [1e30, 3e38])
def test_scale_grows_by_more_than_the_range_of_32_bits(store, chunk, big):
    """The largest finite values after a page's zeros: the scale grows from
    1e-12 / Q to a finite one at most twice what the values need."""
    from cublade_amd.quantization import QuantizedKVCache, append_kv, dequantize_kv
    g = _gen(31)
    cache = QuantizedKVCache.empty(2, 1, 32, 16, store)
    zeros = torch.zeros(3, 1, 32, device=DEV, dtype=torch.bfloat16)
    append_kv(cache, zeros, zeros, _i32([[1]]), _i32([3]), cu_new=_cu([3]))
    n = 2 if chunk else 1
    x = ((torch.rand(n, 1, 32, generator=g, device=DEV) * 2 - 1) * big).bfloat16()
    append_kv(cache, x, x, _i32([[1]]), _i32([3 + n]), cu_new=_cu([n]) if chunk else None)
    q, amax = _kv.QMAX[store], float(x.abs().max())
    for s in (float(cache.k_scale[1]), float(cache.v_scale[1])):
        assert amax / q <= s * (1 + 2.0 ** -22) and s <= 2 * amax / q * (1 + 2.0 ** -22)
    # half a step of the scale (INT8), or of the code (E4M3: 2^-4 relative, and at
    # least 2^-10); a bf16 rounding
    s = float(cache.k_scale[1])
    for t in dequantize_kv(cache, _i32([1])):
        assert bool((t[0, 0, :3] == 0).all())
        want = x[:, 0].double()
        half = s / 2 if store == I8 else (want.abs() * 2.0 ** -4).clamp(min=s * 2.0 ** -10)
        assert bool(((t[0, 0, 3:3 + n].double() - want).abs()
                     <= half * (1 + 2.0 ** -20) + (want.abs() + half) * 2.0 ** -8).all())
