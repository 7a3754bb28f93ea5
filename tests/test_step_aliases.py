"""Results of a drafted step's operators laid over memory that other blocks still read: refused at the C entry points,
with addresses that nobody reads, before anything is launched."""
import ctypes

import pytest

from winnow_b200 import _lib

ADDRESS = 1 << 20


def _keep(out, granted=None):
    """Two sequences: lengths, counts, a path of two and a table row of three at addresses of their own."""
    side = _lib.PoolSide(ADDRESS, ADDRESS, 64, 64, 64, 16, 16, 16, 64)
    return _lib.lib().wtq_keep_tokens(ctypes.byref(side), ctypes.byref(side), 5 * ADDRESS, 3, 2 * ADDRESS, 4 * ADDRESS, 2,
                                      3 * ADDRESS, 1, 2, 2, 16, 4, 3, 2, 4, granted, out, None, None)


@pytest.mark.parametrize("at", [2, 3, 4, 5])
@pytest.mark.parametrize("shift", [-4, 0, 4])
def test_kept_lengths_over_what_is_read(at, shift):
    assert _keep(at * ADDRESS + shift) == -1
    assert b"share memory" in _lib.lib().wtq_last_error()


def test_kept_lengths_over_the_last_words_read():
    assert _keep(4 * ADDRESS + 12) == _keep(5 * ADDRESS + 20) == -1       # the second rows' last entries
    assert _keep(6 * ADDRESS, granted=6 * ADDRESS + 4) == -1
