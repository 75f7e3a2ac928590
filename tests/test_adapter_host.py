"""Low-rank adapters refuse bad arguments before any device work (no GPU needed).

Addresses below are numbers that nothing reads: every call is refused by its checks.
"""
import ctypes as C

import numpy as np
import pytest

from witchcraft_amd import _lib, adapters

P = 1 << 32  # an aligned address
FAR = 1 << 40  # bytes between buffers that do not overlap
LOTS = 1 << 40
lib = _lib.lib


def _refused(fn, *args, says=""):
    rc = fn(*args)
    msg = lib.t5h_last_error().decode()
    assert rc == _lib.T5H_ERR_INVALID, (rc, msg)
    assert says in msg, msg


def _call(x=P, xt=1, xs=None, ldx=128, T=5, K=128, ids=P, G=3, a=P, b=P, wt=1, ranks=None, scales=None, R=16, cols=(64,),
          slices=None, y=P + FAR, ldy=None, out=P + 2 * FAR, ldo=None, yt=1, work=P, bytes_=LOTS):
    n = sum(cols) if cols else 64
    carr = None if cols is None else (C.c_int32 * len(cols))(*cols)
    _call.keep = carr
    return (x, xt, xs, ldx, T, K, ids, G, a, b, wt, ranks, scales, R, None if carr is None else C.addressof(carr),
            len(cols or ()) if slices is None else slices, y, n if ldy is None else ldy, out, n if ldo is None else ldo, yt, work,
            bytes_, None)


@pytest.mark.parametrize("args,says", [
    (dict(T=-1), "rows"), (dict(T=(1 << 30) + 1), "rows"), (dict(K=0), "row length"), (dict(K=100), "row length"),
    (dict(K=(1 << 21) + 16), "row length"), (dict(slices=0), "slices"), (dict(slices=5), "slices"), (dict(R=0), "rank"),
    (dict(R=12), "rank"), (dict(R=136), "rank"), (dict(R=-8), "rank"), (dict(G=-1), "adapters"), (dict(G=(1 << 24) + 1), "adapters"),
    (dict(wt=0), "f16 or bf16"), (dict(wt=3, xt=3), "f16 or bf16"), (dict(xt=2), "type"), (dict(xt=0), "type"), (dict(xt=4), "type"),
    (dict(wt=2, xt=1), "type"), (dict(yt=3), "type of results"), (dict(yt=-1), "type of results"), (dict(cols=None, slices=1), "NULL columns"),
    (dict(cols=(64, 24)), "columns"), (dict(cols=(0,)), "columns"), (dict(cols=(-16, 64)), "columns"), (dict(cols=((1 << 24) + 16,)), "columns"),
    (dict(x=None), "NULL x"), (dict(y=None), "NULL y"), (dict(out=None), "NULL out"), (dict(ids=None), "NULL ids"), (dict(a=None), "NULL a"),
    (dict(b=None), "NULL b"), (dict(work=None), "NULL workspace"), (dict(xt=3), "NULL scales"), (dict(xt=3, xs=P + 8), "scales of x is not aligned"), (dict(xt=3, xs=P, T=1 << 30, K=256), "2^31"), (dict(x=P + 8), "x is not aligned"),
    (dict(y=P + FAR + 4), "y is not aligned"), (dict(out=P + 2), "out is not aligned"), (dict(a=P + 8), "a is not aligned"),
    (dict(b=P + 8), "b is not aligned"), (dict(ids=P + 2), "ids is not aligned"), (dict(ranks=P + 1), "ranks is not aligned"),
    (dict(scales=P + 2), "scales is not aligned"), (dict(work=P + 4), "workspace is not aligned"), (dict(ldx=120), "x's rows"),
    (dict(ldx=132), "x's rows"), (dict(ldx=-128), "x's rows"), (dict(ldx=(1 << 24) + 8), "x's rows"), (dict(ldy=48), "y's rows"),
    (dict(ldo=68), "out's rows"), (dict(ldo=0), "out's rows"), (dict(ldo=(1 << 24) + 8), "out's rows"), (dict(bytes_=5 * 16 * 4 - 1), "workspace is smaller"), (dict(bytes_=0), "workspace"),
    (dict(out=P + FAR + 16), "overlaps"), (dict(out=P + FAR, ldo=128), "overlaps"), (dict(out=P + FAR, ldy=128, ldo=64), "overlaps"),
    # columns of the same rows, which run into the next row's
    (dict(ldy=128, out=P + FAR + 192, ldo=128), "overlaps"), (dict(ldy=128, out=P + FAR + 64, ldo=128), "overlaps"),
])
def test_adapter_add_refuses(args, says):
    _refused(lib.t5h_adapter_add_device, *_call(**args), says=says)


def test_nothing_to_do():
    assert lib.t5h_adapter_add_device(*_call(T=0, x=None, y=None, out=None, work=None)) == 0
    cols = (C.c_int32 * 1)(64)
    assert lib.t5h_adapter_add(0, None, 1, None, 0, 128, None, 3, None, None, 1, None, None, 16, C.addressof(cols), 1, None, None, 1) == 0


def test_workspace():
    assert adapters.workspace_bytes(0, 128, 1, 16) == 0
    for t in (1, 5, 16, 17, 300, 4616, 74640):
        for k in (16, 128, 768, 4096):
            for slices, r in ((1, 8), (3, 16), (4, 128)):
                n = adapters.workspace_bytes(t, k, slices, r)
                assert n >= t * slices * r * 4
    big = adapters.workspace_bytes(1 << 30, 1 << 21, 4, 128)
    assert big == (1 << 30) * 512 * 6
    _refused(lib.t5h_adapter_workspace, 1, 128, 1, 16, None, says="NULL")
    n = C.c_size_t()
    for args, says in (((-1, 128, 1, 16), "rows"), ((1, 8, 1, 16), "row length"), ((1, 128, 5, 16), "slices"), ((1, 128, 1, 4), "rank")):
        _refused(lib.t5h_adapter_workspace, *args, C.byref(n), says=says)


def test_host_form_refuses():
    buf = np.zeros(4096, np.uint8).ctypes.data
    cols = (C.c_int32 * 1)(16)
    c = C.addressof(cols)
    f = lib.t5h_adapter_add
    _refused(f, 0, None, 1, None, 1, 16, buf, 1, buf, buf, 1, None, None, 8, c, 1, buf, buf, 1, says="NULL")
    _refused(f, 0, buf, 3, None, 1, 16, buf, 1, buf, buf, 1, None, None, 8, c, 1, buf, buf, 1, says="NULL")
    _refused(f, 0, buf, 1, None, 1, 16, buf, 1, None, buf, 1, None, None, 8, c, 1, buf, buf, 1, says="NULL")
    _refused(f, 0, buf, 1, None, 1, 20, buf, 1, buf, buf, 1, None, None, 8, c, 1, buf, buf, 1, says="row length")
    _refused(f, 0, buf, 2, None, 1, 16, buf, 1, buf, buf, 1, None, None, 8, c, 1, buf, buf, 1, says="type")


def test_python_checks():
    h = np.float16
    x, ids = np.zeros((4, 128), h), np.zeros(4, np.int32)
    a, b, y = np.zeros((2, 1, 8, 128), h), np.zeros((2, 32, 8), h), np.zeros((4, 32), np.float32)
    for args in ((x[0], ids, a, b, y), (x.astype(np.float32), ids, a, b, y), (x, ids[:2], a, b, y), (x, ids + 0.5, a, b, y),
                 (x, ids, a[0], b, y), (x, ids, a.astype(np.float32), b, y), (x, ids, a[:1], b, y), (x, ids, a[:, :, :4], b, y),
                 (x[:, :64], ids, a, b, y), (x, ids, a, b, y[:, :16]), (x, ids, a, b, y.astype(np.float64)), (x, ids, a[:, :0], b, y),
                 ((x, x), ids, a, b, y), ((np.zeros((4, 128), np.uint8), np.zeros((1, 4), np.uint8)), ids, a, b, y)):
        with pytest.raises(ValueError):
            adapters.add(*args)
    for bad in (dict(scales=np.ones(3)), dict(ranks=[1]), dict(cols=(16,)), dict(cols=(16, 16))):
        with pytest.raises(ValueError):
            adapters.add(x, ids, a, b, y, **bad)
    with pytest.raises(_lib.T5HError, match="rank"):
        adapters.add(x, ids, a[:, :, :4], b[:, :, :4], y)


@pytest.mark.parametrize("size", [1 << 32, -(1 << 32), 1 << 31, -1])
def test_sizes_that_32_bits_do_not_hold(size):
    def device(**kw):
        d = dict(xt=1, T=0, K=128, G=3, wt=1, R=16, yt=1, cols=(64,), ldx=128, ldy=64, ldo=64, bytes_=0)
        d.update(kw)
        adapters.add_device(P, d["xt"], 0, d["ldx"], d["T"], d["K"], P, d["G"], P, P, d["wt"], 0, 0, d["R"], d["cols"], P, d["ldy"], P, d["ldo"],
                            d["yt"], P, d["bytes_"])
    device()
    for name in ("xt", "T", "K", "G", "wt", "R", "yt"):
        with pytest.raises(ValueError, match="2\\^31"):
            device(**{name: size})
    with pytest.raises(ValueError, match="2\\^31"):
        device(cols=(size,))
    for name in ("ldx", "ldy", "ldo", "bytes_"):
        with pytest.raises(ValueError, match="2\\^63"):
            device(**{name: 1 << 64})
    for i in range(4):
        args = [1, 128, 1, 16]
        args[i] = size
        with pytest.raises(ValueError, match="2\\^31"):
            adapters.workspace_bytes(*args)
