"""What the attention's error bound of tests/_kv_tight.py accepts and rejects,
on the CPU: the mistakes are planted in the 64-bit form."""
from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from tests import _kv, _kv_tight

I8, F8 = torch.int8, torch.float8_e4m3fn


def _case(n, new, d, page, store, dt, spread=1.0, hkv=1, rep=2):
    g = torch.Generator().manual_seed(n + d)
    table, pages = _kv.make_table([n], page, g, device="cpu")
    q = _kv.QMAX[store]

    def codes(*shape):
        x = (torch.randn(shape, generator=g) * q / 4).clamp(-q, q)
        return (x.round() if store == I8 else x).to(store)

    def scale():
        return 4 / q * torch.exp2((torch.rand(pages, hkv, generator=g) * 2 - 1) * spread)

    cache = SimpleNamespace(k=codes(pages, hkv, page, d), v=codes(pages, hkv, d, page), k_scale=scale(),
                            v_scale=scale(), kv_heads=hkv, head_dim=d, page_size=page)
    return torch.randn(new, hkv * rep, d, generator=g).to(dt), cache, table


def _block(a, b):
    """Values of the 64 keys from `a` read from `b` (None: lost)."""
    def change(_, v):
        v = v.clone()
        v[:, a:a + 64] = 0 if b is None else v[:, b:b + 64]
        return v
    return change


@pytest.mark.parametrize("store,dt", [(I8, torch.bfloat16), (F8, torch.float16)])
@pytest.mark.parametrize("n,new,d,page", [(9000, 2, 128, 64), (20001, 5, 64, 16), (2500, 40, 128, 32),
                                          (300, 30, 96, 16)])
def test_lost_or_doubled_block_of_values_is_rejected(n, new, d, page, store, dt):
    q, cache, table = _case(n, new, d, page, store, dt)
    ref = _kv_tight.attend_tight(q, cache, table, [n], [new])
    # the kernel's own rounding of the weights is accepted, with room
    got = (ref[4].to(dt), ref[1].float())
    assert _kv_tight.excess(got, ref, dt) <= 1
    for a, b in ((64 * (n // 128 - 2), None), (0, None), (64, 0), (64 * (n // 64 - 2), 0)):
        bad = _kv_tight.attend_tight(q, cache, table, [n], [new], change=_block(a, b))
        assert _kv_tight.excess((bad[0].to(dt), ref[1].float()), ref, dt) > 1, (a, b)


def test_scales_far_apart_keep_the_bound_of_each_page():
    """Value scales 2^20 apart: the bound follows the page that a row's output
    comes from, and the weights' rounding stays within it."""
    q, cache, table = _case(400, 3, 64, 16, I8, torch.float16, spread=20.0)
    ref = _kv_tight.attend_tight(q, cache, table, [400], [3], scale=1e-8)
    assert _kv_tight.excess((ref[4].to(torch.float16), ref[1].float()), ref, torch.float16) <= 1
    # the whole bound is a small part of the values' own size
    assert bool((ref[2] <= 2.0 ** -9 * (ref[0].abs() + ref[0].abs().amax(-1, keepdim=True))).all())
