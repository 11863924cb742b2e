"""A bound on attend_kv's error that does not grow with the number of keys the
way n roundings of the largest value would: what each key can add is bounded by
its own weight. Device-independent (a cache is anything with its tensors and
sizes), so that the CPU can check what the bound rejects.

With s_j the scores, v_j = c_j V_j (code and page scale), y_j = s_j log2 e +
log2 V_j, M its maximum over the visible keys, u_j = 2^(y_j - M), L = sum_j u_j
/ V_j, p_j = u_j / V_j / L: o = sum_j u_j c_j / L. The kernel's errors, each
relative to the term it enters unless said otherwise:
  e_j  of a weight through its exponent: the d products and sums of the score
       ((d + 8) 2^-24 of their magnitudes); a bf16 query element's rounding to
       fp16 under its row's power of two (2^-25 of the row's maximum); three
       roundings of the factor and one of y (2^-24 of s, of y - M, of log V;
       the hardware's log2 and 2^x: one unit in the last place, 2^-23)
  2^-11        a weight's rounding to fp16, in the products only
  2^-25 |c_j|  absolute, for weights below fp16's normal range: relative to a
       running maximum that is never above M, so only where u_j < 2^-14 (2^-13
       here, for the error of u_j)
  A 2^-24      sums over keys in fp32: at most one rounding for 8 keys of a
       matrix product, one or two for each raised maximum (a step of 64), those
       that join waves and ranges: A = n / 8 + 128
  2^-21        1 / L and its product
"""
from __future__ import annotations

import math

import torch

from tests._kv import values, pages_for


def _per_token(x, table, b, length, page):
    """[hkv, length]: a page quantity [pages, hkv] for each token."""
    ids = table[b, :pages_for(length, page)].long()
    return x[ids].double().t().repeat_interleave(page, 1)[:, :length]


def attend_tight(q, cache, table, lens, news, scale=None, causal=True, window=None, change=None):
    """(o, lse, bound on o before its rounding, bound on lse, o with the weights
    rounded to fp16 for its products) in 64 bits. change(b, v): stands in for a
    sequence's values [hkv, n, d] in both o (not in the bound)."""
    t, hq, d = q.shape
    rep = hq // cache.kv_heads
    scale = 1 / math.sqrt(d) if scale is None else scale
    o = torch.zeros(t, hq, d, dtype=torch.float64, device=q.device)
    lse = torch.full((t, hq), -math.inf, dtype=torch.float64, device=q.device)
    bound, lbound = torch.zeros_like(o), torch.zeros_like(lse)
    rounded = torch.zeros_like(o)       # o with the weights rounded as the kernels do
    at = 0
    for b, (n, m) in enumerate(zip(lens, news)):
        if m == 0 or n == 0:
            at += m
            continue
        k, v = values(cache, table, b, n)
        vs = _per_token(cache.v_scale, table, b, n, cache.page_size).clamp(min=2.0 ** -64)
        lv = torch.log(vs)
        v_used = v if change is None else change(b, v)
        key = torch.arange(n, device=q.device)
        pos = n - m + torch.arange(m, device=q.device)
        seen = torch.ones(m, n, dtype=torch.bool, device=q.device)
        if causal:
            seen = key[None] <= pos[:, None]
            if window:
                seen &= key[None] > pos[:, None] - window
        some = seen.any(1)
        sums = n / 8 + 128
        r = slice(at, at + m)
        for h in range(hq):
            g = h // rep
            x = q[r, h].double()
            s = scale * (x @ k[g].t())
            mag = abs(scale) * (x.abs() @ k[g].abs().t())
            few = abs(scale) * x.abs().amax(1, keepdim=True) * k[g].abs().sum(1) * 2.0 ** -25
            y = (s + lv[g]).masked_fill(~seen, -math.inf)              # natural units
            top = torch.where(some, y.amax(1), 0.0)[:, None]
            u = torch.exp(y - top)
            w = u / vs[g]
            big = w.sum(1, keepdim=True).clamp(min=1e-300)
            p = w / big
            e = (mag * (d + 8) * 2.0 ** -24 + few
                 + 2.0 ** -23 * (3 * s.abs() + lv[g].abs() + (y - top).abs().masked_fill(~seen, 0) + 32))
            e = 1.02 * e.masked_fill(~seen, 0)
            pv = p @ v[g].abs()
            pe = (p * e).sum(1, keepdim=True)
            codes = v[g].abs() / vs[g][:, None]
            low = (u < 2.0 ** -13) & seen
            o[r, h] = p @ v_used[g]
            bound[r, h] = (pv * (2.0 ** -11 + sums * 2.0 ** -24) + (p * e) @ v[g].abs()
                           + o[r, h].abs() * (pe + sums * 2.0 ** -24 + 2.0 ** -21)
                           + 2.0 ** -25 * (low.double() @ codes) / big)
            near = u.to(torch.float16).double()
            rounded[r, h] = near @ (v_used[g] / vs[g][:, None]) / big
            lse[r, h] = torch.where(some, torch.logsumexp(s.masked_fill(~seen, -math.inf), 1), -math.inf)
            lbound[r, h] = (pe[:, 0] + sums * 2.0 ** -24
                            + 2.0 ** -22 * (top[:, 0].abs() + torch.log(big[:, 0]).abs() + 16))
        at += m
    return o, lse, bound, lbound, rounded


def excess(got, ref, dtype):
    """Largest error of got (o, lse) in units of its limit: above 1 is wrong."""
    o, lse = got
    ro, rl, bound, lbound = ref[:4]
    ulp = 2.0 ** (-11 if dtype == torch.float16 else -8)
    tiny = 2.0 ** -24 if dtype == torch.float16 else 2.0 ** -126
    over = ((o.double() - ro).abs() / (bound * (1 + ulp) + ro.abs() * ulp + tiny)).max()
    empty = rl == -math.inf
    assert bool((lse[empty] == -math.inf).all())
    if bool(empty.all()):
        return float(over)
    lover = ((lse.double() - rl).abs() / (lbound + rl.abs() * 2.0 ** -23))[~empty].max()
    return max(float(over), float(lover))
