"""linear_w8a8 and gated_w8a8 against plain forms in 64 bits (tests/_w8a8.py)."""
from __future__ import annotations

import pytest
import torch

from tests import _w8a8 as P

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
# rows, output channels, columns: single tokens, both sides of every limit between
# kernels (16, 32, 64 rows), columns that fill no block, no step, no 16 bytes
SHAPES = [(1, 1, 1), (1, 4096, 512), (2, 40, 15), (3, 17, 33), (15, 4100, 272), (16, 9000, 144),
          (17, 100, 1000), (33, 513, 128), (64, 129, 2064), (64, 8200, 130), (65, 128, 64), (65, 1, 16),
          (65, 7, 17), (129, 40, 7), (90, 5000, 784), (128, 11008, 400), (120, 9000, 1001), (129, 70, 33),
          (129, 300, 48), (100, 300, 48), (127, 255, 4096), (128, 256, 272), (257, 511, 1040),
          (300, 1001, 1403), (70, 130, 9), (1000, 520, 640), (2100, 2050, 80), (700, 300, 1001), (640, 1000, 35), (1100, 4100, 531), (260, 4096, 11008)]


def _case(m, n, k, seed, bias, xmode, dtype):
    x, sx = P.codes(m, k, seed)
    w, sw = P.codes(n, k, seed + 1)
    if xmode == "tensor":
        sx = sx[0].clone()
    b = torch.randn(n, generator=torch.Generator().manual_seed(seed + 2)).to(dtype).cuda() if bias else None
    return x, sx, w, sw, b


@pytest.mark.parametrize("i,shape", list(enumerate(SHAPES)))
def test_linear_to_the_last_bit(i, shape):
    from cublade_amd.quantization import linear_w8a8
    dtype = list(DT.values())[i % 3]
    x, sx, w, sw, b = _case(*shape, 10 * i, i % 2 == 0, "tensor" if i % 4 == 3 else "token", dtype)
    y = linear_w8a8(P.qt(x, sx, dtype), P.qt(w, sw), b)
    assert y.dtype == dtype and y.shape == shape[:2]
    want = P.linear(x, sx, w, sw, b, dtype)
    assert torch.equal(y.cpu(), want), (y.cpu().float() - want.float()).abs().max()


@pytest.mark.parametrize("act", P.ACTS)
@pytest.mark.parametrize("shape", [(1, 1, 1), (1, 4100, 528), (5, 33, 17), (16, 9000, 144), (20, 300, 1000),
                                   (64, 70, 130), (65, 128, 64), (90, 129, 33), (128, 64, 4096), (128, 4200, 528), (40, 9000, 777), (33, 13000, 272), (10, 20000, 130),
                                   (129, 129, 33), (140, 64, 4096),
                                   (333, 700, 1400), (700, 300, 1001), (650, 1300, 39), (1030, 1500, 96)])
def test_gated(shape, act):
    from cublade_amd.quantization import gated_w8a8
    m, n, k = shape
    i = P.ACTS.index(act) + m
    dtype = list(DT.values())[i % 3]
    x, sx, g, sg, gb = _case(m, n, k, i, i % 2 == 0, "token", dtype)
    _, _, u, su, ub = _case(1, n, k, i + 7, i % 4 < 2, "token", dtype)
    sx, sg, su = sx * 40 / k ** 0.5, sg / 4, su / 4
    y = gated_w8a8(P.qt(x, sx, dtype), P.qt(g, sg), P.qt(u, su), activation=act, gate_bias=gb, up_bias=ub)
    assert y.dtype == dtype and y.shape == (m, n)
    want, bound = P.gated(x, sx, (g, sg, gb), (u, su, ub), act, dtype)
    err = (y.cpu().double() - want).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


# Sizes that between them take every tile and shape of workgroup: whole, with K cut into
# ranges, with rows of 16 bytes, of words and of any bytes, copied first or not.
LINEAR_FORMS = [
    (954, 16384, 512), (196, 20352, 9984), (1339, 8704, 256), (130, 8881, 9152), (2529, 221, 960),
    (2115, 155, 6032), (242, 5966, 16), (2252, 121, 2832), (218, 214, 16), (935, 204, 16), (316, 1150, 16),
    (364, 746, 688), (921, 640, 640), (760, 1507, 160), (1393, 651, 544), (734, 20635, 268),
    (132, 8995, 10616), (952, 1378, 28), (2145, 106, 6980), (76, 268, 44), (68, 1430, 44), (924, 416, 24),
    (439, 635, 632), (755, 939, 524), (130, 7152, 216), (1853, 450, 556), (385, 31933, 486),
    (7111, 2205, 397), (141, 7955, 8394), (1511, 7743, 186), (2360, 416, 555), (2334, 131, 5274),
    (351, 5388, 25), (2471, 755, 21), (162, 849, 17538), (2222, 111, 2841), (89, 301, 34), (326, 406, 30),
    (100, 3996, 23), (1489, 188, 517), (284, 2154, 569), (952, 1711, 37), (99, 6294, 714),
    (129, 7041, 12032), (19, 102, 16), (33, 5295, 16), (1310, 385, 528), (18, 4098, 16), (17, 6550, 16),
    (541, 393, 16), (1605, 135, 16), (19, 102, 20), (37, 5263, 20), (1176, 281, 524), (18, 4542, 20),
    (33, 4157, 24), (1031, 272, 20), (1076, 150, 1076), (67, 11308, 2307), (17, 114, 17), (40, 2303, 17),
    (17, 4496, 19), (34, 4322, 17), (19, 8352, 17)]
GATED_FORMS = [
    (1255, 6404, 432), (193, 8976, 11376), (825, 5287, 304), (135, 4464, 8272), (749, 1375, 464),
    (67, 3316, 7360), (178, 5645, 16), (65, 5578, 7408), (75, 299, 32), (267, 738, 16), (119, 1388, 528),
    (319, 1665, 160), (338, 776, 768), (129, 30593, 264), (129, 5996, 8636), (142, 3955, 40),
    (133, 903, 13032), (125, 186, 40), (239, 973, 20), (82, 1409, 660), (852, 883, 132), (813, 362, 660),
    (138, 30530, 429), (1235, 6441, 414), (131, 6100, 4211), (1093, 4885, 210), (2356, 179, 1041),
    (893, 159, 12542), (228, 4360, 27), (714, 2173, 22), (88, 389, 13337), (67, 521, 26), (1226, 172, 23),
    (69, 1599, 555), (665, 1263, 39), (1713, 174, 591),
    (138, 4264, 9760), (2226, 107, 2768), (17, 101, 16), (18, 2089, 16), (18, 4816, 2608), (2254, 102,
    1508), (19, 101, 20), (17, 4330, 20), (1087, 129, 24), (65, 100, 14398), (2303, 261, 10515), (20,
    100, 17), (34, 2230, 17)]


@pytest.mark.parametrize("i,shape", list(enumerate(LINEAR_FORMS)))
def test_linear_by_every_form(i, shape):
    test_linear_to_the_last_bit(i + 100, shape)


@pytest.mark.parametrize("i,shape", list(enumerate(GATED_FORMS)))
def test_gated_by_every_form(i, shape):
    test_gated(shape, P.ACTS[i % 4])


@pytest.mark.parametrize("m", [2, 40, 65, 300])
def test_sums_of_the_largest_codes(m):
    """The longest rows of the largest codes, -128 among them: 2^14 K < 2^31."""
    from cublade_amd.quantization import linear_w8a8
    k, n = 131071, 40
    x = torch.full((m, k), -128, dtype=torch.int8, device="cuda")
    w = torch.full((n, k), -128, dtype=torch.int8, device="cuda")
    w[1::2] = 127
    one = torch.ones((), device="cuda")
    y = linear_w8a8(P.qt(x, one), P.qt(w, one), out_dtype=torch.float32)
    assert torch.equal(y.cpu()[0, :2], torch.tensor([k * 16384.0, -k * 16256.0]))
    assert bool((y == y[0]).all()) and bool((y[:, ::2] == y[0, 0]).all())


def test_a_token_does_not_depend_on_its_batch():
    """The same row alone, among few, among many and where K is split: equal bits."""
    from cublade_amd.quantization import gated_w8a8, linear_w8a8
    n, k = 1000, 4096
    x, sx = P.codes(700, k, 1)
    (w, sw), (u, su) = P.codes(n, k, 2), P.codes(n, k, 3)
    sx = sx / 50
    for f in (lambda r: linear_w8a8(P.qt(x[r], sx[r]), P.qt(w, sw)),
              lambda r: gated_w8a8(P.qt(x[r], sx[r]), P.qt(w, sw), P.qt(u, su))):
        whole = f(slice(0, 700))
        for r in (slice(0, 1), slice(3, 20), slice(100, 164), slice(30, 150), slice(200, 330)):
            assert torch.equal(f(r), whole[r])


def test_strided_rows_and_offsets():
    """Codes as columns of a larger tensor, with and without alignment, and scales
    with strides."""
    from cublade_amd.quantization import linear_w8a8
    big, _ = P.codes(800, 640, 5)
    wide, _ = P.codes(96, 512, 6)
    s = torch.rand(1600, device="cuda")[::2] * 0.01
    for m in (3, 64, 128, 200, 800):
        for off, k in ((0, 512), (16, 256), (5, 256), (7, 77), (3, 512)):
            x, w = big[:m, off:off + k], wide[:, :k]
            y = linear_w8a8(P.qt(x, s[:m]), P.qt(w, s[:96]))
            want = P.linear(x, s[:m], w, s[:96], None, torch.float16)
            assert torch.equal(y.cpu(), want), (m, off, k)


def test_offsets_past_32_bits():
    """Codes of more than 2^31 bytes on either side and outputs of more than 2^32: the
    last rows and columns are those of a call on them alone (and of the oracle)."""
    from cublade_amd.quantization import gated_w8a8, linear_w8a8
    g = torch.Generator(device="cuda").manual_seed(3)
    many, few = 1_100_000, 2000
    for k in (2048, 2044):                                # by DMA, and through registers
        big = torch.randint(-127, 128, (many, k), generator=g, device="cuda", dtype=torch.int8)
        sb = torch.rand(many, generator=g, device="cuda") * 0.01
        w, sw = P.codes(few, k, 4)
        tail = slice(many - 70, many)
        small = P.linear(big[tail], sb[tail], w, sw, None, torch.float16)
        y = linear_w8a8(P.qt(big, sb, torch.float16), P.qt(w, sw))
        assert y.numel() * 2 > 1 << 32 and torch.equal(y[tail].cpu(), small)
        y = gated_w8a8(P.qt(big, sb, torch.float16), P.qt(w, sw), P.qt(w, sw), activation="relu")
        ref = gated_w8a8(P.qt(big[tail].contiguous(), sb[tail], torch.float16), P.qt(w, sw), P.qt(w, sw),
                         activation="relu")
        assert torch.equal(y[tail], ref)
        del y
        for m in (3, 20, 70, 300):                        # the large side as the weight
            y = linear_w8a8(P.qt(w[:m], sw[:m], torch.float16), P.qt(big, sb))
            # the product of the scales the other way round: two roundings each
            want = P.sums(w[:m], big[tail]).double() * sw[:m].cpu().double()[:, None] * sb[tail].cpu().double()
            got = y[:, tail].cpu().double()
            # three roundings to fp32 and one to fp16 (normal numbers: the scales see to it,
            # smaller results are within 2^-25)
            assert bool(((got - want).abs() <= want.abs() * (2.0 ** -11 + 3 * 2.0 ** -24) + 2.0 ** -25).all()), m
        del big, y


def test_more_channels_than_a_grid_of_few_rows_takes():
    from cublade_amd.quantization import gated_w8a8, linear_w8a8
    g = torch.Generator(device="cuda").manual_seed(5)
    n, k = (1 << 27) + 40, 16
    w = torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    sw = torch.rand(n, generator=g, device="cuda") * 0.01
    for m in (1, 3):
        x, sx = P.codes(m, k, 6)
        y = linear_w8a8(P.qt(x, sx, torch.float32), P.qt(w, sw))
        u = gated_w8a8(P.qt(x, sx, torch.float32), P.qt(w, sw), P.qt(w, sw), activation="relu")
        for c in (slice(0, 200), slice(1 << 26, (1 << 26) + 200), slice(n - 200, n)):
            want = P.linear(x, sx, w[c], sw[c], None, torch.float32)
            assert torch.equal(y[:, c].cpu(), want)
            assert torch.equal(u[:, c].cpu(), want.clamp(min=0) * want)


def test_less_workspace_gives_the_same():
    """Without a workspace K is not cut and unaligned rows are not copied."""
    import ctypes
    from cublade_amd import _abi
    L = _abi.lib()
    for m, n, k in ((2115, 155, 6032), (2360, 416, 555), (2334, 131, 5274)):
        (x, sx), (w, sw) = P.codes(m, k, 1), P.codes(n, k, 2)
        need = L.cbq_w8a8_ws_bytes(m, n, k, 1)
        assert need > _abi.WS_CTRL_BYTES
        rows = [_abi.I8Rows(q.data_ptr(), k, s.data_ptr(), 1) for q, s in ((x, sx), (w, sw))]
        got = []
        for nbytes in (0, _abi.WS_CTRL_BYTES, need - 1, need):
            y = torch.empty(m, n, device="cuda")
            ws = torch.zeros(max(nbytes, 256), dtype=torch.uint8, device="cuda")
            assert L.cbq_w8a8_linear(ctypes.byref(rows[0]), ctypes.byref(rows[1]), None, 0, m, n, k,
                                     y.data_ptr(), 0, ws.data_ptr() if nbytes else None, nbytes,
                                     _abi.stream_handle(y.device)) == 0
            got.append(y.cpu())
        want = P.linear(x, sx, w, sw, None, torch.float32)
        assert all(torch.equal(y, want) for y in got)


def test_empty_sizes():
    from cublade_amd.quantization import gated_w8a8, linear_w8a8
    for m, n, k in ((0, 8, 16), (4, 0, 16), (4, 8, 0), (80, 8, 0)):
        (x, sx), (w, sw) = P.codes(m, k, 1), P.codes(n, k, 2)
        b = torch.arange(n, dtype=torch.float32, device="cuda") + 0.5
        y = linear_w8a8(P.qt(x, sx), P.qt(w, sw), b)
        assert y.shape == (m, n) and torch.equal(y, b.half().expand(m, n))
        y = gated_w8a8(P.qt(x, sx), P.qt(w, sw), P.qt(w, sw), activation="relu", gate_bias=b, up_bias=b)
        assert torch.equal(y, (b * b).half().expand(m, n))


def test_scales_that_are_not_finite():
    """A NaN scale (a token whose norm was not finite) and an infinite one reach
    their own row or column only."""
    from cublade_amd.quantization import linear_w8a8
    for m in (5, 70):
        (x, sx), (w, sw) = P.codes(m, 128, 1), P.codes(30, 128, 2)
        sx[2], sw[4] = float("nan"), float("inf")
        y = linear_w8a8(P.qt(x, sx), P.qt(w, sw)).cpu()
        want = P.linear(x, sx, w, sw, None, torch.float16)
        assert torch.equal(y.isnan(), want.isnan())
        assert torch.equal(y.nan_to_num(1.0), want.nan_to_num(1.0))
