"""Plain 64-bit forms of the 8-bit paged key/value cache's operators, and cases
of it: a pool with pages in random order, ragged lengths, random codes."""
from __future__ import annotations

import math

import torch

QMAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
DEV = "cuda"


def pages_for(n: int, page: int) -> int:
    return -(-n // page)


def make_table(lens, page, gen, width=None, spare=3, device=DEV):
    """(page_table, number of pages): every sequence's pages in random order
    among the pool's; unused entries hold an id that is not one (-7)."""
    need = [pages_for(n, page) for n in lens]
    total = sum(need) + spare
    order = torch.randperm(total, generator=gen, device=device).to(torch.int32)
    width = width or max(max(need), 1)
    table = torch.full((len(lens), width), -7, dtype=torch.int32, device=device)
    at = 0
    for i, c in enumerate(need):
        table[i, :c] = order[at:at + c]
        at += c
    return table, total


def random_cache(pages, hkv, d, page, store, gen, spread=1.0):
    """A cache of random codes, scales within a factor 4 (times spread)."""
    from cublade_amd.quantization import QuantizedKVCache
    q = QMAX[store]

    def codes(*shape):
        x = (torch.randn(shape, generator=gen, device=DEV) * q / 4).clamp(-q, q)
        return (x.round() if store == torch.int8 else x).to(store)

    def scale():
        e = torch.rand(pages, hkv, generator=gen, device=DEV) * 2 - 1
        return 4 / q * torch.exp2(e * spread)

    return QuantizedKVCache(codes(pages, hkv, page, d), codes(pages, hkv, d, page), scale(), scale())


def values(cache, table, b, length):
    """(k, v) of a sequence in 64 bits, [hkv, length, d]."""
    ids = table[b, :pages_for(length, cache.page_size)].long()
    k = cache.k[ids].double() * cache.k_scale[ids].double()[:, :, None, None]
    v = cache.v[ids].double() * cache.v_scale[ids].double()[:, :, None, None]
    hkv, d = cache.kv_heads, cache.head_dim
    k = k.transpose(0, 1).reshape(hkv, -1, d)[:, :length]
    v = v.permute(1, 0, 3, 2).reshape(hkv, -1, d)[:, :length]
    return k, v


def attend_ref(q, cache, table, lens, news, scale=None, causal=True, window=None):
    """(o, lse, bound on |error| of o before its rounding, of lse) in 64 bits.

    The bound, per output: with p the probabilities,
      sum_j p_j |v_j| (2^-10 + 4 delta) + 127 * 2^-24 * n * max v scale
    2^-11 is one rounding of a weight to fp16 (2^-10 with the sum's own), delta
    bounds the error of a score in fp32: the products' sums, the query's
    rounding to fp16 under a power of two (2^-25 of its row's maximum, per
    element), the exponent's rounding (its size, up to 2 max |s| + 64, times
    2^-23) and n additions; the last term is weights below fp16's normal range
    (2^-25 absolute, against a largest weight of at least 1)."""
    t, hq, d = q.shape
    rep = hq // cache.kv_heads
    scale = 1 / math.sqrt(d) if scale is None else scale
    o = torch.zeros(t, hq, d, dtype=torch.float64, device=q.device)
    lse = torch.full((t, hq), -math.inf, dtype=torch.float64, device=q.device)
    bound, lbound = torch.zeros_like(o), torch.zeros_like(lse)
    at = 0
    for b, (n, m) in enumerate(zip(lens, news)):
        if m == 0:
            continue
        k, v = values(cache, table, b, n)
        key = torch.arange(n, device=q.device)
        pos = n - m + torch.arange(m, device=q.device)
        seen = torch.ones(m, n, dtype=torch.bool, device=q.device)
        if causal:
            seen = key[None] <= pos[:, None]
            if window:
                seen &= key[None] > pos[:, None] - window
        for h in range(hq):
            if n == 0:
                continue
            x = q[at:at + m, h].double()
            kh, vh = k[h // rep], v[h // rep]
            s = scale * (x @ kh.t())
            mag = abs(scale) * (x.abs() @ kh.abs().t())
            rounded = abs(scale) * x.abs().amax(1, keepdim=True) * kh.abs().sum(1) * 2.0 ** -25
            s = s.masked_fill(~seen, -math.inf)
            some = seen.any(1)
            l = torch.logsumexp(s, 1)
            p = torch.where(some[:, None], torch.exp(s - l[:, None]), 0.0)
            p = torch.where(seen, p, 0.0)
            delta = (mag * (d + 8) * 2.0 ** -24 + rounded
                     + (2 * s.masked_fill(~seen, 0).abs().amax(1, keepdim=True) + 64) * 2.0 ** -23
                     + n * 2.0 ** -24)
            delta = delta.masked_fill(~seen, 0).amax(1)
            r = slice(at, at + m)
            o[r, h] = torch.where(some[:, None], p @ vh, 0.0)
            vmax = float(vh.abs().max()) if n else 0.0
            bound[r, h] = (p @ vh.abs()) * (2.0 ** -10 + 4 * delta)[:, None] + 2.0 ** -24 * n * vmax
            lse[r, h] = l
            lbound[r, h] = 2 * delta + 2.0 ** -20
        at += m
    return o, lse, bound, lbound


def assert_attends(got, ref, dtype, what=""):
    """got (o, lse) against attend_ref's result, with one rounding of o."""
    o, lse = got
    ro, rl, bound, lbound = ref
    ulp = 2.0 ** (-11 if dtype == torch.float16 else -8)
    tiny = 2.0 ** -24 if dtype == torch.float16 else 0.0
    err = (o.double() - ro).abs()
    limit = bound * (1 + ulp) + ro.abs() * ulp + tiny
    assert bool((err <= limit).all()), (what, float((err / limit.clamp(min=1e-30)).max()))
    empty = rl == -math.inf
    assert bool((lse[empty] == -math.inf).all()), what
    err = (lse.double() - rl).abs()[~empty]
    assert bool((err <= (lbound + rl.abs() * 2.0 ** -23)[~empty]).all()), (what, "lse")


def rotate_ref(x, pos, cos, sin, interleaved):
    """x [tokens, heads, d] turned to the tables' rows pos, in 64 bits."""
    x = x.double().clone()
    half = cos.shape[1]
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
    i = torch.arange(half, device=x.device)
    i1, i2 = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    a, b = x[..., i1], x[..., i2]
    x[..., i1], x[..., i2] = a * c - b * s, b * c + a * s
    return x


def rotate_f32(x, pos, cos, sin, interleaved):
    """The same with every product and sum rounded to 32 bits."""
    x = x.float().clone()
    half = cos.shape[1]
    c, s = cos[pos][:, None], sin[pos][:, None]
    i = torch.arange(half, device=x.device)
    i1, i2 = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    a, b = x[..., i1].clone(), x[..., i2].clone()
    x[..., i1], x[..., i2] = a * c - b * s, b * c + a * s
    return x


def tables(rows, rot, device=DEV):
    half = rot // 2
    ang = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (
        -torch.arange(half, dtype=torch.float64) / half)
    return ang.cos().float().to(device), ang.sin().float().to(device)


def encode(x, store):
    if store == torch.int8:
        return torch.nan_to_num(torch.round(x), nan=0.0).clamp(-127, 127).to(torch.int8)
    return x.clamp(-448, 448).to(store)


class CacheModel:
    """What append_kv does, token block by token block, in fp32 torch
    operations: the same formulas, so codes and scales have to be equal."""

    def __init__(self, cache):
        self.store, self.page = cache.dtype, cache.page_size
        self.k, self.v = cache.k.clone(), cache.v.transpose(2, 3).contiguous()
        self.ks, self.vs = cache.k_scale.clone(), cache.v_scale.clone()

    def put(self, x, codes, scale, table_row, first):
        """x fp32 [tokens, hkv, d] at positions first ..."""
        q = QMAX[self.store]
        n = x.shape[0]
        for p in range(first // self.page, pages_for(first + n, self.page)):
            lo, hi = max(first, p * self.page), min(first + n, (p + 1) * self.page)
            pid, off = int(table_row[p]), lo - p * self.page
            new = x[lo - first:hi - first].transpose(0, 1)             # [hkv, tokens, d]
            amax = torch.nan_to_num(new.abs(), nan=0.0, posinf=math.inf).amax((1, 2))
            s = scale[pid]
            if off == 0:
                inv = torch.full_like(amax, q) / amax.clamp(min=1e-12)   # one rounding
                s_new = 1 / inv
            else:
                ratio = amax / (q * s)
                mant, e = torch.frexp(ratio)
                g = torch.where(ratio > 1, torch.where(mant > 0.5, e, e - 1), 0)
                s_new = torch.ldexp(s, g)
                old = torch.ldexp(codes[pid, :, :off].float(), -g[:, None, None])
                codes[pid, :, :off] = encode(old, self.store)
                inv = 1 / s_new
            codes[pid, :, off:off + hi - lo] = encode(new * inv[:, None, None], self.store)
            scale[pid] = s_new

    def append(self, k, v, table, lens, news):
        at = 0
        for b, (n, m) in enumerate(zip(lens, news)):
            if m:
                row = table[b].tolist()
                self.put(k[at:at + m], self.k, self.ks, row, n - m)
                self.put(v[at:at + m].float(), self.v, self.vs, row, n - m)
            at += m

    def assert_equal(self, cache, what=""):
        def same(a, b):
            return bool((a.view(torch.uint8) == b.view(torch.uint8)).all())
        assert same(self.ks, cache.k_scale) and same(self.vs, cache.v_scale), (what, "scales")
        assert same(self.k, cache.k), (what, "k")
        assert same(self.v, cache.v.transpose(2, 3).contiguous()), (what, "v")
