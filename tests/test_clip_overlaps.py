"""Clipped gradients that overlap in memory are refused before HIP is touched: two
workgroups would write, or read and write, the same elements in any order."""
from array import array

import pytest

from novann_amd import _lib

A = 0x100000  # never dereferenced: every refused call below fails validation first
F32, BF16, F64 = 0, 2, 6


def clip(rows, workspace=1 << 30):
    """The status of rows (grad, out, n, grad's type, out's type)."""
    table = array("q")
    for grad, out, n, gdt, odt in rows:
        table.extend([grad, out, n, gdt | odt << 32])
    return _lib.load().novaq_clip_grad_norm(table.buffer_info()[0], len(rows), 1.0, 0.0, A, A,
                                            workspace, None)


@pytest.mark.parametrize("rows", [
    [(A, A, 100, F32, F32), (A, A, 100, F32, F32)],                  # one gradient twice
    [(A, A, 100, F32, F32), (A + 160, A + 160, 100, F32, F32)],      # overlapping views
    [(A + 160, A + 160, 10, F32, F32), (A, A, 100, F32, F32)],       # one inside another
    [(A, A + 4000, 100, F32, F32), (A + 4000, A, 100, F32, F32)],    # into each other
    [(A, A + 4000, 100, F32, F32), (A + 8000, A + 4396, 100, F32, F32)],  # outputs overlap
    [(A, A + 16, 100, F32, F32)],                                    # shifted in place
    [(A, A, 100, BF16, F32)],                                        # widened in place
    [(A, A, 100, F64, F32)],
    [(A, 0, 100, F32, F32), (A + 4000, A + 4000, 8, F32, F32), (A + 4028, A + 4028, 8, F32, F32)],
    [(A + 1000 * i, A + 1000 * i, 250, F32, F32) for i in range(300)]
    + [(A + 4, A + 4, 1, F32, F32)],                                 # the list past the stack's
])
def test_refused(rows):
    assert clip(rows) == _lib.EINVAL


def test_sizes_past_the_address_space_are_refused():
    assert clip([(A, A, 1 << 62, F32, F32)]) == _lib.EINVAL
