"""Sizes past which the loops of a drafted step's kernels would leave 32 bits: refused at the C entry points, with
addresses that nobody reads."""
import ctypes

import pytest

from winnow_b200 import _lib

AT = 1 << 40
FAR = 1 << 36                                  # apart from one another at any of the sizes below


def _plan(tokens, stack):
    out = _lib.Plan(*(AT + (10 + i) * FAR for i in range(9)))
    return _lib.lib().wtq_plan_tokens(AT, AT + FAR, None, 0, AT + 2 * FAR, 4, AT + 3 * FAR, AT + 4 * FAR, AT + 5 * FAR, 3, 4, 16,
                                      tokens, 0, stack, ctypes.byref(out), None, None, None)


@pytest.mark.parametrize("tokens,stack", [((1 << 30) + 1, 5), (2 ** 31 - 1, 5), (9, (1 << 30) + 1), (9, 2 ** 31 - 1)])
def test_plans_beyond_32_bits(tokens, stack):
    assert _plan(tokens, stack) == -1
    assert b"2^30" in _lib.lib().wtq_last_error()


def test_releases_beyond_32_bits():
    assert _lib.lib().wtq_release_tokens(AT, AT + FAR, 4, AT + 2 * FAR, AT + 3 * FAR, AT + 4 * FAR, AT + 5 * FAR, 2, 4,
                                         (1 << 30) + 1, None, None) == -1
