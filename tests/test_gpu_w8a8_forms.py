"""Products in the forms that the sizes of tests/test_gpu_w8a8.py do not choose: each case
names its form and fails where its sizes no longer choose it. The check that no form is left
out is tests/test_w8a8_forms_host.py."""
from __future__ import annotations

import pytest

from tests import _w8a8 as P
from tests import _w8a8_forms as F
from tests import test_gpu_w8a8 as T

pytestmark = pytest.mark.gpu

# form (tests/_w8a8_forms.py), sizes
LINEAR = [
    (("few", 16, 16, 512, 1, 4, True), (1, 1, 20)), (("few", 16, 16, 512, 1, 4, True), (13, 700, 1004)),
    (("few", 32, 16, 512, 1, 1, True), (1, 4976, 17)), (("few", 32, 16, 512, 1, 16, True), (2, 4215, 1120)),
    (("few", 32, 16, 512, 1, 4, True), (1, 4366, 1080)), (("few", 32, 64, 512, 1, 1, False), (1614, 165, 17)),
    (("few", 48, 16, 512, 1, 1, True), (1, 9676, 17)), (("few", 48, 16, 512, 1, 4, True), (1, 11659, 20)),
    (("few", 64, 16, 256, 1, 1, True), (1, 14568, 21)), (("few", 64, 16, 256, 1, 16, True), (1, 13370, 16)),
    (("few", 64, 16, 256, 1, 4, True), (1, 14412, 20)), (("few", 64, 32, 256, 1, 16, False), (79, 4106, 16)),
    (("tiles", 256, 192, 2, 1, True, "copies"), (829, 2444, 16565)),
    (("tiles", 256, 256, 2, 1, True, "copies"), (1542, 2760, 13209)),
    (("short", 1), (300, 50, 15)),
]
GATED = [
    (("few", 32, 16, 512, 2, 4, True), (1, 1, 20)), (("few", 32, 16, 512, 2, 4, True), (16, 333, 2044)),
    (("few", 64, 16, 256, 2, 4, True), (1, 4462, 20)), (("few", 96, 16, 512, 2, 1, False), (22, 4141, 559)),
    (("few", 96, 16, 512, 2, 1, True), (1, 9181, 622)), (("few", 96, 16, 512, 2, 16, False), (20, 4246, 12464)),
    (("few", 96, 16, 512, 2, 16, True), (1, 11008, 4096)), (("few", 96, 16, 512, 2, 16, True), (1, 8695, 2528)),
    (("few", 96, 16, 512, 2, 4, True), (1, 9827, 11796)),
    (("tiles", 256, 192, 2, 2, True, "copies"), (956, 2049, 8758)),
    (("tiles", 256, 256, 2, 2, True, "copies"), (907, 2367, 13209)),
    (("short", 2), (70, 90, 3)),
]


@pytest.mark.parametrize("i", range(len(LINEAR)))
def test_linear(i):
    form, shape = LINEAR[i]
    assert F.key(*shape, 1) == form
    T.test_linear_to_the_last_bit(i + 200, shape)


@pytest.mark.parametrize("i", range(len(GATED)))
def test_gated(i):
    form, shape = GATED[i]
    assert F.key(*shape, 2) == form
    for act in (P.ACTS if i % 4 == 0 else (P.ACTS[i % 4],)):
        T.test_gated(shape, act)
