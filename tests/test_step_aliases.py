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


NAMES = [n for n, _ in _lib.Plan._fields_]
ORDER = ("lengths", "new", "in_held", "free", "in_count", "parents", "table", *NAMES)


def _at(name, shift=0):
    return (2 + ORDER.index(name)) * ADDRESS + shift


def _plan(tree=False, ticket=None, **at):
    """Three sequences of up to four pages, nine tokens (trees of three), five free pages, each at an address of its own."""
    place = {**{n: _at(n) for n in ORDER}, **at}
    out = _lib.Plan(*(place[n] for n in NAMES))
    return _lib.lib().wtq_plan_tokens(place["lengths"], None if tree else place["new"], place["parents"] if tree else None, 3,
                                      place["table"], 4, place["in_held"], place["free"], place["in_count"], 3, 4, 16, 9,
                                      3 if tree else 0, 5, ctypes.byref(out), ticket, None, None)


@pytest.mark.parametrize("out", NAMES[:8])
@pytest.mark.parametrize("over", ["lengths", "new", "in_held", "free", "in_count", "table"])
def test_planned_results_over_what_is_read(out, over):
    own = {"seq_lens": "lengths", "held": "in_held", "free_count": "in_count"}.get(out)
    if own != over:
        assert _plan(**{out: _at(over)}, ticket=99 * ADDRESS) == -1
    if over != "in_count" and out != "free_count":
        assert _plan(**{out: _at(over, 4)}, ticket=99 * ADDRESS) == -1       # a shifted view of it, their own state among it
    assert b"share memory" in _lib.lib().wtq_last_error()


@pytest.mark.parametrize("i", range(8))
def test_planned_results_over_one_another(i):
    for j in range(i):
        assert _plan(**{NAMES[i]: _at(NAMES[j])}, ticket=99 * ADDRESS) == -1
    assert _plan(tree=True, mask=_at(NAMES[i])) == -1


def test_planned_results_over_the_trees_and_the_ticket():
    assert _plan(tree=True, positions=_at("parents", 32)) == _plan(tree=True, table=_at("parents")) == -1
    assert _plan(tree=True, mask=_at("parents", -32)) == -1
    assert _plan(seq_lens=_at("lengths"), ticket=_at("starts", 8)) == -1
    assert b"share memory" in _lib.lib().wtq_last_error()
