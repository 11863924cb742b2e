"""One scale for a whole weight, scales with strides, and biases of other types than the
output's, by each kind of kernel: one output per thread, few rows, tiles, K in ranges."""
from __future__ import annotations

import pytest
import torch

from tests import _w8a8 as P
from tests import _w8a8_forms as F

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.mark.parametrize("m,n,k,kernel,cut", [(5, 40, 9, F.SHORT, False), (7, 300, 528, F.FEW, False),
                                              (2360, 416, 555, F.TILES, False), (2304, 256, 11008, F.TILES, True)])
@pytest.mark.parametrize("out,bias", [(F32, F16), (F16, F32), (BF16, F16), (F16, BF16)])
def test_scales_and_biases(m, n, k, kernel, cut, out, bias):
    from cublade_amd.quantization import gated_w8a8, linear_w8a8
    for projections in (1, 2):
        f = F.form(m, n, k, projections)
        assert f.kernel == kernel and (f.ranges > 1) == cut
    (x, sx), (w, sw), (u, su) = (P.codes(r, k, s) for r, s in ((m, 1), (n, 2), (n, 3)))
    wide = torch.zeros(2 * n, device="cuda")
    wide[::2] = su / 4
    scales = (sx * 40 / k ** 0.5, sw[0] / 4, wide[::2])
    b, c = (torch.randn(n, generator=torch.Generator().manual_seed(s)).to(bias).cuda() for s in (4, 5))
    for s in (scales[1], scales[2]):
        y = linear_w8a8(P.qt(x, scales[0]), P.qt(w, s), b, out_dtype=out)
        assert torch.equal(y.cpu(), P.linear(x, scales[0], w, s, b, out))
    for act, gb, ub in (("silu", b, None), ("gelu_tanh", None, c), ("relu", b, c)):
        y = gated_w8a8(P.qt(x, scales[0]), P.qt(w, scales[1]), P.qt(u, scales[2]), activation=act, gate_bias=gb,
                       up_bias=ub, out_dtype=out)
        want, bound = P.gated(x, scales[0], (w, scales[1], gb), (u, scales[2], ub), act, out)
        assert bool(((y.cpu().double() - want).abs() <= bound).all())
