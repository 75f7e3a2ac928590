"""Head norms and rotation: the table of frequencies, and bad arguments refused before any device work (no GPU needed).

Addresses below are numbers that nothing reads: every call is refused by its checks.
"""
from fractions import Fraction

import numpy as np
import pytest

from witchcraft_amd import _lib, rotary

P = 1 << 32  # an aligned address
FAR = 1 << 36  # bytes between buffers that do not overlap
PI = Fraction("3.14159265358979323846264338327950288419716939937510")


def _refused(fn, *args, says=""):
    rc = fn(*args)
    msg = _lib.lib.t5h_last_error().decode()
    assert rc == _lib.T5H_ERR_INVALID, (rc, msg)
    assert says in msg, msg


# ---- the table -----------------------------------------------------------------------------

@pytest.mark.parametrize("freqs", [
    [1.0, 0.5, 1e-3, 1e-9, 0.0, -1.0, -1e-300, 1e-300, 5e-324, 6.283185307179586, 12345.678, -0.25, 2.0 ** 40 + 0.5],
    list(10000.0 ** (-np.arange(64) / 64)), list(1e6 ** (-np.arange(128) / 128))])
def test_table_holds_turns(freqs):
    """Entries are within half a step of 2^-61 of the frequency in turns modulo 1; the division's own rounding,
    2^-64 of the turns, adds to that for those above one turn."""
    got = rotary.table(freqs)
    for f, e in zip(freqs, got.tolist()):
        assert e & 7 == 0
        turns = Fraction(f) / (2 * PI)
        d = (Fraction(e >> 3, 1 << 61) - turns) % 1
        assert min(d, 1 - d) <= Fraction(1, 1 << 62) + abs(turns) * Fraction(3, 1 << 64), (f, e)


def test_table_holds_axes():
    axes = [0, 1, 2, 7, 3, 0]
    got = rotary.table([0.1] * 6, axes)
    assert (got & np.uint64(7)).tolist() == axes
    assert (got >> np.uint64(3) == rotary.table([0.1])[0] >> np.uint64(3)).all()
    assert rotary.table([]).shape == (0,)


def test_table_refuses():
    t, f, a = (np.zeros(300, x) for x in (np.uint64, np.float64, np.int32))
    call = _lib.lib.t5h_rotary_table
    _refused(call, f.ctypes.data, None, -1, t.ctypes.data, says="pairs")
    _refused(call, f.ctypes.data, None, 257, t.ctypes.data, says="pairs")
    _refused(call, None, None, 4, t.ctypes.data, says="NULL")
    _refused(call, f.ctypes.data, None, 4, None, says="NULL")
    for v in (np.nan, np.inf, -np.inf):
        f[3] = v
        _refused(call, f.ctypes.data, None, 4, t.ctypes.data, says="finite")
    f[3] = 0
    for v in (-1, 8):
        a[2] = v
        _refused(call, f.ctypes.data, a.ctypes.data, 4, t.ctypes.data, says="axis")
    for bad in (dict(axes=[0.5, 0.0]), dict(axes=[0]), dict(axes=[0, 8]), dict(axes=[0, 1 << 32])):
        with pytest.raises(ValueError):
            rotary.table([1.0, 0.5], **bad)
    with pytest.raises(ValueError):
        rotary.table([[1.0]])


def test_frequencies():
    f = rotary.frequencies(8, 10000.0)
    assert f.dtype == np.float64 and np.allclose(f, [1.0, 0.1, 0.01, 0.001], rtol=1e-15)


# ---- refusals ------------------------------------------------------------------------------

def _call(q=P, ldq=256, qh=2, k=P + FAR, ldk=128, kh=1, t=1, T=5, D=128, qg=None, kg=None, eps=1e-6, table=P, rot=128,
          pairing=0, pos=P, axes=1, qo=P + 2 * FAR, ldqo=256, ko=P + 3 * FAR, ldko=128):
    return q, ldq, qh, k, ldk, kh, t, T, D, qg, kg, eps, table, rot, pairing, pos, axes, qo, ldqo, ko, ldko, None


@pytest.mark.parametrize("args,says", [
    (dict(T=-1), "rows"), (dict(T=(1 << 30) + 1), "rows"), (dict(qh=-1), "heads"), (dict(kh=65536), "heads"),
    (dict(D=0), "head size"), (dict(D=-8), "head size"), (dict(D=100), "head size"), (dict(D=520), "head size"),
    (dict(rot=-8), "rotated"), (dict(rot=136), "rotated"), (dict(rot=60), "rotated"), (dict(t=3), "type"),
    (dict(t=-1), "type"), (dict(pairing=2), "pairing"), (dict(pairing=-1), "pairing"), (dict(axes=0), "axes"),
    (dict(axes=9), "axes"), (dict(eps=-1e-6), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"),
    (dict(q=None), "NULL q"), (dict(k=None), "NULL k"), (dict(qo=None), "NULL q_out"), (dict(ko=None), "NULL k_out"),
    (dict(table=None), "NULL"), (dict(pos=None), "NULL"), (dict(table=P + 4), "table"), (dict(pos=P + 2), "positions"),
    (dict(qg=P + 2), "gammas"), (dict(kg=P + 1), "gammas"), (dict(q=P + 8), "q's rows"), (dict(ko=P + 8), "k_out's rows"),
    (dict(ldq=260), "q's rows"), (dict(ldq=248), "as long as"), (dict(ldko=120), "as long as"), (dict(ldq=-256), "as long as"),
    (dict(ldq=(1 << 30) + 8), "as long as"), (dict(ldqo=0), "as long as"),
    # outputs over inputs that are not their own, or only in part, or with other row lengths
    (dict(qo=P + 16), "overlaps"), (dict(qo=P, ldqo=264), "overlaps"), (dict(ko=P + FAR - 16), "overlaps"),
    (dict(ko=P), "overlaps"), (dict(qo=P + FAR + 128), "overlaps"), (dict(ko=P + 2 * FAR), "overlaps"),
    # columns of one projection's rows: k's results reach into the next row's q
    (dict(ldq=512, k=P + 512, ldk=512, qo=P, ldqo=512, ko=P + 800, ldko=512), "overlaps"),
    (dict(ldq=512, k=P + 512, ldk=512, qo=P, ldqo=512, ko=P + 1024 - 128, ldko=512), "overlaps"),
])
def test_rotary_refuses(args, says):
    _refused(_lib.lib.t5h_rotary_device, *_call(**args), says=says)


def test_nothing_to_do():
    """No rows or no heads: fine, whatever the buffers."""
    f = _lib.lib.t5h_rotary_device
    assert f(*_call(T=0, q=None, qo=None)) == 0
    assert f(*_call(qh=0, kh=0, q=None, k=3)) == 0
    assert _lib.lib.t5h_rotary(0, None, 2, None, 1, 0, 0, 64, None, None, 1e-6, None, 64, 0, None, 1, None, None) == 0
    q = np.zeros((0, 2, 64), np.float32)
    a, b = rotary.rotate(q, q, np.zeros(0, np.int32), rotary.table(rotary.frequencies(64)))
    assert a.shape == b.shape == (0, 2, 64)


def test_host_form_refuses():
    buf = np.zeros(4096, np.uint8).ctypes.data
    f = _lib.lib.t5h_rotary
    _refused(f, 0, None, 1, buf, 1, 0, 1, 64, None, None, 1e-6, buf, 64, 0, buf, 1, buf, buf, says="NULL")
    _refused(f, 0, buf, 1, buf, 1, 0, 1, 64, None, None, 1e-6, None, 64, 0, buf, 1, buf, buf, says="NULL")
    _refused(f, 0, buf, 1, buf, 1, 0, 1, 60, None, None, 1e-6, buf, 56, 0, buf, 1, buf, buf, says="head size")
    _refused(f, 0, buf, 1, buf, 1, 9, 1, 64, None, None, 1e-6, buf, 64, 0, buf, 1, buf, buf, says="type")


def test_python_checks():
    q, k, tab = np.zeros((3, 2, 64), np.float32), np.zeros((3, 1, 64), np.float32), rotary.table(rotary.frequencies(64))
    pos = np.arange(3)
    for args in ((q[0], k, pos, tab), (q, k.astype(np.float16), pos, tab), (q, k[:2], pos, tab), (q, k[:, :, :32], pos, tab),
                 (q.astype(np.float64), k, pos, tab), (q, k, pos[:2], tab), (q, k, pos.astype(np.float32), tab),
                 (q, k, pos + 2 ** 31, tab), (q, k, pos, tab.astype(np.int64)), (q, k, pos, tab[None])):
        with pytest.raises(ValueError):
            rotary.rotate(*args)
    with pytest.raises(ValueError, match="q_gamma"):
        rotary.rotate(q, k, pos, tab, q_gamma=np.ones(32))
    with pytest.raises(_lib.T5HError, match="rotated"):
        rotary.rotate(q, k, pos, rotary.table(rotary.frequencies(128)))


@pytest.mark.parametrize("size", [1 << 32, -(1 << 32), 1 << 31, -1])
def test_sizes_that_32_bits_do_not_hold(size):
    names = ["qh", "kh", "t", "T", "D", "rot", "pairing", "axes"]
    for name in names:
        args = dict(T=0)
        args[name] = size
        c = list(_call(**args))[:-1]
        c[9], c[10] = 0, 0
        with pytest.raises(ValueError, match="2\\^31"):
            rotary.rotate_device(*c)
    for name in ("ldq", "ldk", "ldqo", "ldko"):
        c = list(_call(T=0, **{name: 1 << 64}))[:-1]
        with pytest.raises(ValueError, match="2\\^63"):
            rotary.rotate_device(*c)
