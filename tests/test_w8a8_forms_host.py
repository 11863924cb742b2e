"""The kernels that W8A8 products of given sizes choose (no GPU work)."""
from __future__ import annotations

import ctypes

import pytest

from tests import _w8a8_forms as F


@pytest.mark.parametrize("projections", [1, 2])
@pytest.mark.parametrize("k", [16, 20, 17, 4096])
def test_grids_have_fewer_than_2_to_32_threads(k, projections):
    """Every accepted number of channels: a launch takes fewer than 2^32 threads."""
    edges = [1 << e for e in range(26, 31)] + [(1 << 31) - 400]
    for n in sorted({max(1, min(e + d, (1 << 31) - 257)) for e in edges for d in (-64, -1, 0, 1, 40, 64, 200)}):
        for m in (1, 3, 16, 17, 64, 65, 256):
            f = F.form(m, n, k, projections)
            assert f.workgroups * f.threads < 1 << 32, (m, n, f.kernel, f.weight_rows, f.workgroups)
            assert f.workgroups * f.weight_rows // projections >= n     # every channel has an owner


def test_sizes_that_no_grid_takes_are_refused():
    """M N past what tiles of 256 x 256 cover: a workspace size, and an error from a call."""
    from cublade_amd import _abi
    L = _abi.lib()
    big = (1 << 30) + 1
    assert L.cbq_w8a8_ws_bytes(big, big, 64, 1) >= _abi.WS_CTRL_BYTES
    rows = _abi.I8Rows(4096, 64, 4096, 1)
    for f in (lambda: L.cbq_w8a8_linear(ctypes.byref(rows), ctypes.byref(rows), None, 0, big, big, 64, 4096, 1,
                                        None, 0, None),
              lambda: L.cbq_w8a8_gated(ctypes.byref(rows), ctypes.byref(rows), ctypes.byref(rows), None, None, 0, 0,
                                       big, big, 64, 4096, 1, None, 0, None)):
        assert f() == 1 and "too many tiles" in L.cbq_last_error().decode()


def test_bad_arguments_of_the_query():
    from cublade_amd import _abi
    L = _abi.lib()
    f = _abi.W8A8Form()
    for args, needle in (((0, 8, 64, 1, 16), "sizes"), ((8, 0, 64, 1, 16), "sizes"), ((8, 8, 131072, 1, 16), "sizes"),
                         ((8, 8, 64, 3, 16), "projections"), ((8, 8, 64, 1, 8), "multiple"),
                         ((8, 8, 63, 1, 4), "multiple")):
        assert L.cbq_w8a8_form_of(*args, ctypes.byref(f)) == 1 and needle in L.cbq_last_error().decode()
    assert L.cbq_w8a8_form_of(8, 8, 64, 1, 16, None) == 1
    assert F.form(8, 8, 7, 1).kernel == F.SHORT


def test_every_form_is_among_the_cases():
    """The forms that random sizes choose are those that some case of the GPU tests has: a
    change of the choice shows here where it leaves a kernel without a test."""
    import random
    from tests import test_gpu_w8a8 as T
    from tests import test_gpu_w8a8_forms as N
    gated = next(m for m in T.test_gated.pytestmark if m.args[0] == "shape").args[1]
    for cases in (N.LINEAR, N.GATED):
        for form, shape in cases:
            assert F.key(*shape, form[1] if form[0] == "short" else form[4]) == form, shape
    tested = {F.key(*s, 1) for s in T.SHAPES + T.LINEAR_FORMS} | {F.key(*s, 2) for s in gated + T.GATED_FORMS}
    tested |= {form for form, _ in N.LINEAR + N.GATED}
    rng = random.Random(1)

    def size(lo, hi):
        return round(2 ** rng.uniform(lo, hi))

    for _ in range(60000):
        m, n, k, projections = size(0, 12), size(0, 15.3), size(3.5, 14.3), rng.choice((1, 2))
        rows = rng.choice((1, 4, 16))
        k = max(rows, k // rows * rows)
        assert F.key(m, n, k, projections) in tested, (m, n, k, projections)
