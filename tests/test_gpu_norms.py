"""norm_tensor and residual_norm against plain forms in 64 bits (tests/_norms.py)."""
from __future__ import annotations

import pytest
import torch

from tests import _norms as P

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _rand(*shape, seed, dtype=F32, spread=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * spread + shift).to(dtype)


def _gpu(*ts):
    return [None if t is None else t.cuda() for t in ts]


# every kernel: a wave per row (one and two chunks), a workgroup (one, two and four
# chunks), rows read again; few and many tokens; sizes that end inside a chunk
HIDDEN = [1, 2, 7, 8, 64, 500, 512, 513, 1000, 1403, 2048, 4096, 5120, 8192, 8200, 16384, 20000,
          32768, 33001]


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("hidden", HIDDEN)
def test_norm(hidden, kind):
    from cublade_amd.quantization import norm_tensor
    i = HIDDEN.index(hidden)
    dtype, out = (F32, F16, BF16)[i % 3], (torch.int8, F32, F16, BF16, torch.int8)[i % 5]
    for tokens in ((1, 5) if hidden > 9000 else (1, 3, 700)):
        x = _rand(tokens, hidden, seed=i, dtype=dtype, shift=0.3)
        if hidden == 1 and kind == "layer":
            x = torch.zeros_like(x)      # a single element is its own mean
        w = _rand(hidden, seed=i + 50, spread=0.3, shift=1.0, dtype=dtype) if i % 4 else None
        b = _rand(hidden, seed=i + 60, dtype=dtype) if (i + (kind == "layer")) % 2 else None
        for to in {out, torch.int8}:
            got = norm_tensor(*_gpu(x, w, b), kind=kind, eps=1e-5, dtype=to)
            y, err = P.norm(x.double(), torch.zeros(x.shape, dtype=torch.float64), kind, 1e-5, w, b)
            if to is torch.int8:
                assert got.data.shape == x.shape and got.scale.shape == (tokens,)
                assert got.original_dtype == dtype
                P.check_codes(got.data, got.scale, y, err)
            else:
                assert got.dtype == to and got.shape == x.shape
                off = (got.cpu().double() - y).abs()
                bound = (err + P.half(to) * y.abs()) * 1.01 + P.tiny(to)
                assert bool((off <= bound).all()), float((off / bound).max())


GATES = [None, "channel", "token", "full", "scalar"]


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("hidden", [3, 64, 505, 1024, 1403, 4096, 8192, 16384, 30000, 33001])
def test_residual(hidden, post):
    from cublade_amd.quantization import residual_norm
    for j in range(2 if hidden > 9000 else 4):
        i = 10 * hidden + j
        tokens = (2, 5, 600, 9)[j]
        kind = ("rms", "layer")[(j // 2 + post) % 2]
        xt = (F16, BF16, F32, BF16)[(hidden + j) % 4]
        rt = xt if j % 2 == 0 else F32
        pt = xt if j % 3 else F32                            # parameters
        gate = GATES[(hidden + j) % 5]
        x = _rand(tokens, hidden, seed=i, dtype=xt, spread=2.0)
        r = _rand(tokens, hidden, seed=i + 1, dtype=rt, spread=3.0)
        w, b, pw, pb = (_rand(hidden, seed=i + 2 + k, dtype=pt, spread=0.3, shift=k % 2 == 0) for k in range(4))
        if not post:
            pw = pb = None
        if kind == "rms":
            b = None
        g = None if gate is None else _rand(
            *{"channel": (hidden,), "token": (tokens, 1), "full": (tokens, hidden), "scalar": (1,)}[gate],
            seed=i + 9, dtype=(xt, F32)[j % 2])
        alpha = (1.0, 0.25, -1.5, 0.1)[j]
        out = (torch.int8, xt, torch.int8, BF16)[j]
        h, n = residual_norm(*_gpu(x, r, w, b), kind=kind, eps=1e-6, dtype=out, post_norm=post,
                             post_weight=_gpu(pw)[0], post_bias=_gpu(pb)[0], gate=_gpu(g)[0], scale=alpha)
        want, bound = P.residual(x, r, kind, 1e-6, post, pw, pb, g, alpha, rt)
        assert h.dtype == rt and h.shape == r.shape
        off = (h.cpu().double() - want).abs()
        assert bool((off <= bound).all()), float((off / bound).max())
        y, err = P.norm(h.cpu().double(), torch.zeros_like(want), kind, 1e-6, w, b)
        if out is torch.int8:
            P.check_codes(n.data, n.scale, y, err)
            assert n.original_dtype == xt
        else:
            off = (n.cpu().double() - y).abs()
            bound = (err + P.half(out) * y.abs()) * 1.01 + P.tiny(out)
            assert n.dtype == out and bool((off <= bound).all()), float((off / bound).max())
        # h alone, and the norm of h in a call of its own: equal bits
        h2, none = residual_norm(*_gpu(x, r), kind=kind, eps=1e-6, dtype=None, post_norm=post,
                                 post_weight=_gpu(pw)[0], post_bias=_gpu(pb)[0], gate=_gpu(g)[0],
                                 scale=alpha)
        assert none is None and torch.equal(h2, h)


def test_norm_of_the_stored_residual_equals_its_own_call():
    from cublade_amd.quantization import norm_tensor, residual_norm
    for hidden in (100, 1000, 4096, 8192):
        x, r, w = _gpu(_rand(40, hidden, seed=1, dtype=BF16), _rand(40, hidden, seed=2, dtype=BF16),
                       _rand(hidden, seed=3, dtype=BF16))
        h, n = residual_norm(x, r, w)
        m = norm_tensor(h, w)
        assert torch.equal(n.data, m.data) and torch.equal(n.scale, m.scale)


def test_codes_read_back_and_feed_a_product():
    from cublade_amd.quantization import dequantize_tensor, linear_w8a8, norm_tensor, quantize_tensor
    x, = _gpu(_rand(3, 20, 512, seed=4, dtype=F16))
    q = norm_tensor(x)
    assert q.data.shape == (60, 512)
    w = quantize_tensor(_rand(64, 512, seed=5, dtype=F16).cuda(), mode="channel")
    y = linear_w8a8(q, w)
    want = dequantize_tensor(q).double() @ dequantize_tensor(w).double().t().contiguous()
    # both values rounded to fp16 in `want`: 2^-11 each of every product's magnitude
    mag = dequantize_tensor(q).double().abs() @ dequantize_tensor(w).double().abs().t().contiguous()
    assert y.dtype == F16 and bool(((y.double() - want).abs() <= mag * 2.0 ** -9).all())


def test_rows_with_nan_and_infinity():
    """Such a token is NaN (its scale, and with it whatever is read back); the
    others are as without it."""
    from cublade_amd.quantization import dequantize_tensor, norm_tensor, residual_norm
    for hidden in (64, 1000, 1403, 4096, 40000):
        for kind in ("rms", "layer"):
            x = _rand(6, hidden, seed=6, dtype=BF16)
            clean = norm_tensor(x.cuda(), kind=kind)
            x[1, hidden // 2], x[3, 0], x[4, hidden - 1] = float("nan"), float("inf"), -float("inf")
            q = norm_tensor(x.cuda(), kind=kind)
            bad = torch.tensor([False, True, False, True, True, False])
            assert torch.equal(q.scale.cpu().isnan(), bad)
            assert torch.equal(q.data[~bad], clean.data[~bad]) and torch.equal(q.scale[~bad], clean.scale[~bad])
            assert bool(dequantize_tensor(q)[bad].isnan().all())
            h, n = residual_norm(x.cuda(), torch.zeros_like(x).cuda(), kind=kind)
            assert torch.equal(h.cpu().isnan(), x.isnan()) and torch.equal(n.scale.cpu().isnan(), bad)


def test_rows_of_zeros_and_of_one_value():
    from cublade_amd.quantization import norm_tensor
    x = torch.zeros(3, 500, dtype=F16, device="cuda")
    x[1] = 2.5
    for kind in ("rms", "layer"):
        q = norm_tensor(x, kind=kind)
        assert int(q.data[0].abs().max()) == 0 and bool(torch.isfinite(q.scale).all())
        y = norm_tensor(x, kind=kind, dtype=F32)
        assert bool((y[0] == 0).all())
        assert bool(((y[1] - (1 if kind == "rms" else 0)).abs() <= 1e-5).all())


def test_views_are_read_in_place():
    """Rows that are slices of wider ones, odd offsets (which another kernel takes, with
    the sums in another order), one row with a stride of its own, transposed input."""
    from cublade_amd.quantization import norm_tensor, residual_norm
    big = _rand(30, 1500, seed=7, dtype=F16).cuda()
    for x in (big[:, 3:1003], big[::2, 100:612], big[4:5, 1:78], big[:, :64].t(), big[3],
              big.view(5, 6, 1500)[:, 2], big[:, 1:65], big[:, 2:1026]):
        rows = x.cpu().reshape(-1, x.shape[-1])
        zero = torch.zeros(rows.shape, dtype=torch.float64)
        a = norm_tensor(x)
        P.check_codes(a.data, a.scale, *P.norm(rows.double(), zero, "rms", 1e-6, None, None))
        h, n = residual_norm(x, x, gate=x)
        want, bound = P.residual(rows, rows, "rms", 1e-6, False, None, None, rows, 1.0, F16)
        assert h.shape == x.shape
        stored = h.cpu().double().reshape(rows.shape)
        assert bool(((stored - want).abs() <= bound).all())
        P.check_codes(n.data, n.scale, *P.norm(stored, zero, "rms", 1e-6, None, None))


def test_more_tokens_than_a_launch_takes():
    """2^21 tokens to a launch: tokens on both sides of the border and at the end."""
    from cublade_amd.quantization import norm_tensor, residual_norm
    m, hidden = 2 * (1 << 21) + 5, 8
    g = torch.Generator(device="cuda").manual_seed(8)
    x, r = (torch.randn(m, hidden, generator=g, device="cuda") for _ in range(2))
    gate = torch.rand(m, 1, generator=g, device="cuda")
    q = norm_tensor(x)
    h, n = residual_norm(x, r, gate=gate, dtype=F32)
    zero = torch.zeros(64, hidden, dtype=torch.float64)
    for at in (0, (1 << 21) - 32, (1 << 22) - 60, m - 64):
        c = slice(at, at + 64)
        P.check_codes(q.data[c], q.scale[c], *P.norm(x[c].cpu().double(), zero, "rms", 1e-6, None, None))
        want, bound = P.residual(x[c].cpu(), r[c].cpu(), "rms", 1e-6, False, None, None,
                                 gate[c].cpu().expand(64, hidden), 1.0, F32)
        stored = h[c].cpu().double()
        assert bool(((stored - want).abs() <= bound).all())
        want, bound = P.norm(stored, zero, "rms", 1e-6, None, None)
        assert bool(((n[c].cpu().double() - want).abs() <= bound + want.abs() * 2.0 ** -24).all())


def test_offsets_past_32_bits():
    """More than 2^32 bytes of every tensor: the last tokens are those of their own call
    with as many tokens as make it the same kernel."""
    from cublade_amd.quantization import residual_norm
    for m, hidden in ((300_000, 8192), (1_600_000, 1403)):
        g = torch.Generator(device="cuda").manual_seed(9)
        x = torch.randn(m, hidden, generator=g, device="cuda", dtype=BF16)
        gate = torch.rand(m, hidden, generator=g, device="cuda", dtype=BF16)
        h, n = residual_norm(x, x, gate=gate, dtype=BF16)
        t = slice(m - 1000, m)
        h2, n2 = residual_norm(x[t], x[t], gate=gate[t], dtype=BF16)
        assert x.numel() * 2 > 1 << 32 and torch.equal(h[t], h2) and torch.equal(n[t], n2)
        want, bound = P.residual(x[t].cpu(), x[t].cpu(), "rms", 1e-6, False, None, None, gate[t].cpu(), 1.0, BF16)
        assert bool(((h2.cpu().double() - want).abs() <= bound).all())
        del x, gate, h, n


def test_small_values_without_eps():
    """eps = 0: the mean square of 2^-64 is 2^-128, a denormal; rows of one value, so the
    sums are exact and the norm is 1 up to the division's, the root's and the product's
    roundings (each at most 2^-23)."""
    from cublade_amd.quantization import norm_tensor
    for hidden in (64, 1000, 8192, 40000):
        x = torch.full((3, hidden), 2.0 ** -64, device="cuda")
        y = norm_tensor(x, eps=0.0, dtype=F32)
        # 1 / hidden is rounded, and a denormal sum to 2^-149: 2^-21 of 2^-128
        assert bool(((y - 1).abs() <= 3 * 2.0 ** -23 + 2.0 ** -21).all()), float((y - 1).abs().max())


def test_empty_and_refusals_on_the_gpu():
    from cublade_amd.quantization import norm_tensor, residual_norm
    e = torch.zeros(0, 64, dtype=F16, device="cuda")
    q = norm_tensor(e)
    assert q.data.shape == (0, 64) and q.scale.shape == (0,)
    h, n = residual_norm(e, e, gate=torch.ones(64, device="cuda"), dtype=F16)
    assert h.shape == n.shape == (0, 64)
    assert norm_tensor(torch.zeros(4, 0, device="cuda")).data.shape == (4, 0)
    x = torch.zeros(4, 64, dtype=F16, device="cuda")
    w = torch.ones(64, device="cuda")
    for kw, needle in ((dict(weight=w[:63]), "weight"), (dict(weight=w, bias=w.half()), "one dtype"),
                       (dict(weight=w.double()), "weight"), (dict(kind="batch"), "kind"),
                       (dict(dtype=torch.int32), "dtype"), (dict(weight=w.cpu()), "weight")):
        with pytest.raises(RuntimeError, match=needle):
            norm_tensor(x, **kw)
    for args, kw, needle in (((x, x[:3]), {}, "residual"), ((x, x.bfloat16()), {}, "residual"),
                             ((x, x), dict(gate=w[:5]), "broadcast"), ((x, x), dict(post_weight=w), "post_norm"),
                             ((x, x), dict(gate=w.cpu()), "gate"), ((x.int(), x), {}, "float32")):
        with pytest.raises(RuntimeError, match=needle):
            residual_norm(*args, **kw)
