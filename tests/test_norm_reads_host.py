"""What layer_norm reads of rows that start anywhere, by the arithmetic that its kernels use (no GPU): each row whole, and nothing
outside the tensor."""
import ctypes

import pytest


def ranges(rows, d):
    from asrn_b200 import _lib
    L, lo, hi = _lib.lib(), ctypes.c_int64(), ctypes.c_int64()
    for row in range(rows):
        assert L.asrn_test_norm_reads(rows, d, row, ctypes.addressof(lo), ctypes.addressof(hi)) == 0
        yield row, lo.value, hi.value


@pytest.mark.parametrize('d', [*range(1, 32), 77, 257, 333, 431, 1017, 1025, 2047, 5001, 16377])
def test_nothing_outside_the_tensor(d):
    for rows in (*range(1, 34), 119):
        for row, lo, hi in ranges(rows, d):
            assert 0 <= lo <= row * d and lo % 8 == 0 and row * d - lo < 8, (rows, row)
            assert (row + 1) * d <= hi <= rows * d, (rows, row)


def test_refusals():
    from asrn_b200 import _lib
    L, at = _lib.lib(), ctypes.addressof(ctypes.c_int64())
    f = L.asrn_test_norm_reads
    assert f(4, 3, 4, at, at) == 1 and f(4, 3, -1, at, at) == 1 and f(4, 0, 0, at, at) == 1 and f(4, 3, 0, None, at) == 1
