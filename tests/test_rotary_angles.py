"""How near the rotation's angles are to position * frequency, over all 32-bit positions (no GPU needed).

The kernel multiplies the table's 61-bit fraction of a turn by the position, modulo a turn, and keeps the upper 32 bits
of the fraction; here the same in whole numbers, against exact fractions.  An entry is off by half a step of 2^-61 and by
the division's rounding, 3 x 2^-64 of the turns; the cut takes less than 2^-32 off.  Up to one turn a step that is
(7 x 2^-64) 2^31 + 2^-32 = 9 x 2^-33 turns at the farthest position, which is below 2^-27 radians.
"""
from fractions import Fraction

import numpy as np
import pytest

from witchcraft_amd import rotary

TWO_PI = 2 * Fraction("3.14159265358979323846264338327950288419716939937510")
POSITIONS = [0, 1, -1, 4095, -4096, 131071, 1 << 20, (1 << 24) + 1, 1999999973, -1500000001, 2 ** 31 - 1, -2 ** 31, 2 ** 31 - 2, -2 ** 31 + 1]


def _off(entry, frequency, position):
    """Radians between the kernel's angle and the exact one, the shorter way round."""
    kept = (entry & ~7) * position % (1 << 64) >> 32
    d = (Fraction(kept, 1 << 32) - Fraction(frequency) * position / TWO_PI) % 1
    return min(d, 1 - d) * TWO_PI


@pytest.mark.parametrize("name,freqs", [
    ("ladder of 10,000", rotary.frequencies(128)), ("ladder of 1,000,000", rotary.frequencies(256, 1e6)),
    ("ladder of 500,000, heads of 80", rotary.frequencies(80, 5e5)),
    ("about a turn", [6.283185307179586, 6.283185307179587, 6.28, -6.283185307179586, 3.141592653589793, 2.0, -1.0]),
    ("small", [1e-9, -1e-9, 1e-300, -1e-300, 5e-324, 0.0, 2.0 ** -61])])
def test_up_to_one_turn_a_step(name, freqs):
    worst = max(_off(e, float(f), p) for f, e in zip(freqs, rotary.table(freqs).tolist()) for p in POSITIONS)
    assert worst <= Fraction(1, 1 << 27), float(worst * 2 ** 29)


@pytest.mark.parametrize("frequency", [7.0, 100.0, -12345.678, 1e6, 2.0 ** 40 + 0.5, 1e12])
def test_more_than_one_turn_a_step(frequency):
    """Each further turn a step adds up to 2^-28 radians at the farthest position."""
    entry = rotary.table([frequency]).tolist()[0]
    turns = abs(Fraction(frequency)) / TWO_PI
    for p in POSITIONS:
        assert _off(entry, frequency, p) <= Fraction(1, 1 << 27) + turns * Fraction(abs(p), 1 << 59), p
