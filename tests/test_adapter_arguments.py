"""What witchcraft_amd.adapters takes for ids and ranks, and .rotary for positions, ahead of any device work (no GPU needed).

The library's call is replaced by one that keeps what it is given.
"""
import ctypes as C

import numpy as np
import pytest

from witchcraft_amd import adapters, rotary


def _taken(monkeypatch, module, name, at, n):
    """What the call's array argument `at` of n int32 holds, while it lasts."""
    seen = []

    class Library:
        pass

    setattr(Library, name, staticmethod(lambda *args: seen.extend((C.c_int32 * n).from_address(args[at])) or 0))
    monkeypatch.setattr(module, "lib", Library)
    return seen


def _inputs(t=4, g=2):
    h = np.float16
    return (np.zeros((t, 128), h), np.zeros(t, np.int32), np.zeros((g, 1, 8, 128), h), np.zeros((g, 32, 8), h), np.zeros((t, 32), np.float32))


@pytest.mark.parametrize("ranks", [[7.9, 3.2], [8.0, 4.0], np.array([8, 8], np.float32), [True, False], [8, 0.5], ["8", "8"], [8 + 0j, 8]])
def test_ranks_that_are_not_whole(ranks):
    """Refused, as ids are: a rank that is cut to a whole one would drop or add values in silence."""
    with pytest.raises(ValueError, match="ranks must be whole numbers"):
        adapters.add(*_inputs(), ranks=ranks)


@pytest.mark.parametrize("ranks,want", [([8, 3], [8, 3]), ([99, -5], [8, 0]), (np.array([2 ** 40, -2 ** 40]), [8, 0]),
                                        (np.array([2 ** 63 + 5, 1], np.uint64), [8, 1]), (np.array([5, 255], np.uint8), [5, 8]),
                                        (np.array([-128, 127], np.int8), [0, 8])])
def test_ranks_that_are_whole(monkeypatch, ranks, want):
    """Of any type and size, those outside 0 .. R as the nearer of both."""
    seen = _taken(monkeypatch, adapters, "t5h_adapter_add", 11, 2)
    adapters.add(*_inputs(), ranks=ranks)
    assert seen == want


def test_no_rows_and_no_adapters():
    """Empty lists, which numpy takes for floats, are no fractions."""
    x, ids, a, b, y = _inputs(t=0)
    assert adapters.add(x, [], a, b, y).shape == (0, 32)
    assert adapters.add(x, ids, a[:0], b[:0], y, ranks=[], scales=[]).shape == (0, 32)


def test_no_positions():
    q, tab = np.zeros((0, 2, 64), np.float32), rotary.table(rotary.frequencies(64))
    for none in ([], [[], []], np.zeros((3, 0))):
        a, b = rotary.rotate(q, q, none, tab)
        assert a.shape == b.shape == (0, 2, 64)
    with pytest.raises(ValueError, match="positions"):
        rotary.rotate(q, q, [0.5], tab)
