"""Products with more channels than the grids of few rows take: they go by tiles, and past
2^30 gated channels by the larger of them (2^24 workgroups of 256 threads are too many)."""
from __future__ import annotations

import pytest
import torch

from tests import _w8a8 as P
from tests import _w8a8_forms as F

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,tile", [((1 << 29) + 40, 128), ((1 << 30) + 64, 256)])
def test_channels_past_2_to_29(n, tile):
    from cublade_amd.quantization import gated_w8a8, linear_w8a8
    g = torch.Generator(device="cuda").manual_seed(7)
    k = 16
    w = torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    sw = torch.rand(n, generator=g, device="cuda") * 0.01
    at = [slice(0, 200), slice(n // 2 - 100, n // 2 + 100), slice((1 << 29) - 100, (1 << 29) + 40), slice(n - 200, n)]
    for m in (1, 2):
        f = F.form(m, n, k, 2)
        assert f.kernel == F.TILES and f.weight_rows == tile
        x, sx = P.codes(m, k, 6)
        y = linear_w8a8(P.qt(x, sx, torch.float32), P.qt(w, sw))
        u = gated_w8a8(P.qt(x, sx, torch.float32), P.qt(w, sw), P.qt(w, sw), activation="relu")
        for c in at:
            want = P.linear(x, sx, w[c], sw[c], None, torch.float32)
            assert torch.equal(y[:, c].cpu(), want)
            assert torch.equal(u[:, c].cpu(), want.clamp(min=0) * want)
        del y, u
