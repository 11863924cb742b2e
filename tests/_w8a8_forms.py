"""What a W8A8 product launches (cbq_w8a8_form_of), for tests that name a kernel: they fail
where the sizes no longer choose it, instead of testing another one."""
from __future__ import annotations

import ctypes

SHORT, FEW, TILES = 0, 1, 2


def form(m: int, n: int, k: int, projections: int, multiple: int | None = None):
    """multiple None: rows without padding, at addresses that K's multiple divides."""
    from cublade_amd import _abi
    if multiple is None:
        multiple = 16 if k % 16 == 0 else 4 if k % 4 == 0 else 1
    f = _abi.W8A8Form()
    _abi.check(_abi.lib().cbq_w8a8_form_of(m, n, k, projections, multiple, ctypes.byref(f)), "form")
    return f


def workspace(m: int, n: int, k: int, projections: int) -> int:
    """Bytes past the control block that a call asks for."""
    from cublade_amd import _abi
    return _abi.lib().cbq_w8a8_ws_bytes(m, n, k, projections) - _abi.WS_CTRL_BYTES


def key(m: int, n: int, k: int, projections: int):
    """What tells one form from another: the kernel with its template's choices, and whether K is
    cut and rows are copied first. Rows without padding."""
    f = form(m, n, k, projections)
    rows = 16 if k % 16 == 0 else 4 if k % 4 == 0 else 1
    if f.kernel == SHORT:
        return ("short", projections)
    if f.kernel == FEW:     # up to 16 rows of x: workgroups in their own order
        return ("few", f.weight_rows, f.x_rows, f.threads, projections, rows, f.x_rows == 16 and m <= 16)
    return ("tiles", f.weight_rows, f.x_rows, f.stages, projections, f.ranges > 1, "copies" if f.copies else rows)
