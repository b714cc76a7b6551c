"""What the row kernels read of rows off 16-byte boundaries (csrc/rows.cuh), worked out on the host by
the kernels' own rule for every row and every lane of the warps that hold it: nothing outside the
tensor, and every element."""
import ctypes

import pytest

from hp_rms_norm_b200 import capi


def reads(rows, hidden, stride, start):
    """(elements before the tensor, elements behind it, vectors with an element not read)"""
    out = (ctypes.c_int64 * 3)(-1, -1, -1)
    assert capi.load().hprn_test_loose_reads(rows, hidden, stride, start, out) == capi.OK
    return tuple(out)


@pytest.mark.parametrize("start", range(8))
@pytest.mark.parametrize("rows", [1, 2, 3, 9, 40])
def test_reads_stay_inside_the_tensor(rows, start):
    for hidden in range(1, 521):
        for pad in (0, 1, 3, 7, 8, 13, 300):
            assert reads(rows, hidden, hidden + pad, start) == (0, 0, 0), (hidden, pad)


@pytest.mark.parametrize("hidden", [1001, 2731, 5001, 8191, 16383])
def test_long_rows(hidden):
    for start in range(8):
        for rows in (1, 2, 17):
            assert reads(rows, hidden, hidden, start) == (0, 0, 0)


def test_refusals():
    out = (ctypes.c_int64 * 3)()
    for bad in ((0, 8, 8, 0), (1, 0, 8, 0), (1, 8, 7, 0), (1, 8, 8, 8), (1, 8, 8, -1), (1 << 20, 8, 8, 0)):
        assert capi.load().hprn_test_loose_reads(*bad, out) == capi.ERR_INVALID_ARGUMENT
    assert capi.load().hprn_test_loose_reads(1, 8, 8, 0, None) == capi.ERR_INVALID_ARGUMENT
