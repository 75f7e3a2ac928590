"""The 8-bit operators refuse bad arguments before any device work (no GPU needed).

Addresses below are numbers that nothing reads: every call is refused by its checks.
"""
import numpy as np
import pytest

from witchcraft_amd import _lib, fp8

P = 1 << 20  # an aligned address
BIG = (1 << 30) + 16


def _refused(fn, *args, says=""):
    rc = fn(*args)
    msg = _lib.lib.t5h_last_error().decode()
    assert rc == _lib.T5H_ERR_INVALID, (rc, msg)
    assert says in msg, msg


@pytest.mark.parametrize("x,t,m,k,codes,scales,says", [
    (P, 0, -1, 128, P, P, "rows"), (P, 0, BIG, 128, P, P, "rows"), (P, 0, 4, 0, P, P, "row length"),
    (P, 0, 4, (1 << 21) + 16, P, P, "row length"), (P, 0, 4, 24, P, P, "row length"), (P, 0, 4, -128, P, P, "row length"), (P, 0, 4, BIG, P, P, "row length"),
    (P, 3, 4, 128, P, P, "type"), (P, -1, 4, 128, P, P, "type"), (None, 0, 4, 128, P, P, "NULL"),
    (P, 0, 4, 128, None, P, "NULL"), (P, 0, 4, 128, P, None, "NULL"), (P + 4, 0, 4, 128, P, P, "aligned"),
    (P, 0, 4, 128, P + 8, P, "aligned"), (P, 0, 4, 128, P, P + 1, "aligned"), (P, 0, 1 << 30, 512, P, P, "blocks"),
])
def test_quantize_refuses(x, t, m, k, codes, scales, says):
    _refused(_lib.lib.t5h_fp8_quantize_device, x, t, m, k, codes, scales, None, says=says)


@pytest.mark.parametrize("w,t,n,k,st,codes,scales,says", [
    (P, 0, -1, 128, 0, P, P, "rows"), (P, 0, 4, 8, 0, P, P, "row length"), (P, 9, 4, 128, 0, P, P, "type"),
    (P, 0, 4, 128, 2, P, P, "scale type"), (P, 0, 4, 128, -1, P, P, "scale type"), (None, 0, 4, 128, 0, P, P, "NULL"),
    (P, 0, 4, 128, 0, P + 2, P, "aligned"), (P, 0, 4, 128, 1, P, P + 2, "aligned"), (P, 0, 4, 128, 0, P, None, "NULL"),
])
def test_quantize_weights_refuses(w, t, n, k, st, codes, scales, says):
    _refused(_lib.lib.t5h_fp8_quantize_weights_device, w, t, n, k, st, codes, scales, None, says=says)


def _norm(x=P, xt=0, delta=None, dt=0, m=4, d=128, gamma=P, eps=1e-6, total=None, codes=P, scales=P):
    return x, xt, delta, dt, m, d, gamma, eps, total, codes, scales, None


@pytest.mark.parametrize("args,says", [
    (dict(m=-1), "rows"), (dict(d=100), "row length"), (dict(xt=3), "type"), (dict(delta=P * 4, dt=5), "type"),
    (dict(eps=-1e-6), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"),
    (dict(total=P * 3), "delta"), (dict(x=None), "NULL"), (dict(gamma=None), "NULL"), (dict(codes=None), "NULL"),
    (dict(scales=None), "NULL"), (dict(gamma=P + 4), "aligned"), (dict(delta=P * 4 + 2, dt=1), "aligned"),
    (dict(delta=P * 4, total=P * 3 + 4), "aligned"),
    (dict(delta=P * 4, total=P + 16), "overlaps x"),             # a part of x
    (dict(delta=P * 4, dt=1, total=P * 4), "overlaps delta"),    # f32 sums over an f16 delta
    (dict(delta=P * 4, total=P * 4 - 32), "overlaps delta"),
])
def test_rmsnorm_refuses(args, says):
    _refused(_lib.lib.t5h_fp8_rmsnorm_device, *_norm(**args), says=says)


def _product(a=P, a_s=P, m=4, w=P, w_s=P, n=32, k=128, st=0, c=P, ct=0):
    return a, a_s, m, w, w_s, n, k, st, c, ct, None


@pytest.mark.parametrize("args,says", [
    (dict(m=-1), "rows"), (dict(n=-1), "rows"), (dict(n=BIG), "rows"), (dict(k=40), "row length"),
    (dict(k=(1 << 21) + 16), "row length"), (dict(st=7), "scale type"), (dict(ct=3), "type"), (dict(a=None), "NULL"), (dict(a_s=None), "NULL"),
    (dict(w=None), "NULL"), (dict(w_s=None), "NULL"), (dict(c=None), "NULL"), (dict(a=P + 1), "aligned"),
    (dict(a_s=P + 8), "aligned"), (dict(w=P + 8), "aligned"), (dict(st=1, w_s=P + 1), "aligned"),
    (dict(c=P + 4), "aligned"),
])
def test_matmul_refuses(args, says):
    _refused(_lib.lib.t5h_fp8_matmul_device, *_product(**args), says=says)


def _gated(a=P, a_s=P, m=4, w0=P, w0s=P, w1=P, w1s=P, n=32, k=128, st=0, codes=P, scales=P):
    return a, a_s, m, w0, w0s, w1, w1s, n, k, st, codes, scales, None


@pytest.mark.parametrize("args,says", [
    (dict(n=40), "columns"), (dict(m=-1), "rows"), (dict(k=16 * 5 + 1), "row length"), (dict(st=2), "scale type"),
    (dict(w1=None), "NULL"), (dict(w1s=None), "NULL"), (dict(codes=None), "NULL"), (dict(scales=None), "NULL"),
    (dict(w1=P + 4), "aligned"), (dict(st=1, w1s=P + 2), "aligned"), (dict(scales=P + 4), "aligned"),
    (dict(m=1 << 29, n=1024), "blocks"),
])
def test_gated_gelu_refuses(args, says):
    _refused(_lib.lib.t5h_fp8_gated_gelu_device, *_gated(**args), says=says)


def test_nothing_to_do():
    """No rows or no columns: fine, whatever the buffers."""
    lib = _lib.lib
    assert lib.t5h_fp8_quantize_device(None, 0, 0, 128, None, None, None) == 0
    assert lib.t5h_fp8_quantize_weights_device(None, 0, 0, 128, 0, None, None, None) == 0
    assert lib.t5h_fp8_rmsnorm_device(*_norm(x=None, m=0, codes=None)) == 0
    assert lib.t5h_fp8_matmul_device(*_product(a=None, m=0)) == 0
    assert lib.t5h_fp8_matmul_device(*_product(w=None, n=0)) == 0
    assert lib.t5h_fp8_gated_gelu_device(*_gated(a=None, m=0)) == 0
    assert lib.t5h_fp8_quantize(0, None, 0, 0, 128, None, None) == 0
    assert lib.t5h_fp8_matmul(0, None, None, 0, None, None, 3, 128, 0, None, 0) == 0


def test_host_forms_refuse():
    lib = _lib.lib
    buf = np.zeros(4096, np.uint8).ctypes.data
    _refused(lib.t5h_fp8_quantize, 0, buf, 0, 4, 100, buf, buf, says="row length")
    _refused(lib.t5h_fp8_quantize, 0, None, 0, 4, 128, buf, buf, says="NULL")
    _refused(lib.t5h_fp8_quantize_weights, 0, buf, 0, 4, 128, 3, buf, buf, says="scale type")
    _refused(lib.t5h_fp8_rmsnorm, 0, buf, 0, None, 0, 1, 128, buf, 1e-6, buf, buf, buf, says="delta")
    _refused(lib.t5h_fp8_matmul, 0, buf, buf, 1, buf, buf, 1, 128, 0, buf, 4, says="type")
    _refused(lib.t5h_fp8_gated_gelu, 0, buf, buf, 1, buf, buf, buf, buf, 24, 128, 0, buf, buf, says="columns")


def test_python_checks():
    x = np.zeros((4, 128), np.float32)
    codes, scales = np.zeros((4, 128), np.uint8), np.zeros((1, 16), np.uint8)
    wc, ws = np.zeros((32, 128), np.uint8), np.zeros((1, 1), np.uint8)
    for bad in (x[0], x.astype(np.float64)):
        with pytest.raises(ValueError):
            fp8.quantize(bad)
        with pytest.raises(ValueError):
            fp8.quantize_weights(bad)
    with pytest.raises(ValueError, match="gamma"):
        fp8.rmsnorm(x, np.ones(64, np.float32))
    with pytest.raises(ValueError, match="delta"):
        fp8.rmsnorm(x, np.ones(128, np.float32), delta=x[:2])
    with pytest.raises(ValueError, match="scales"):
        fp8.matmul((codes, scales[:, :4]), (wc, ws))
    with pytest.raises(ValueError, match="scales"):
        fp8.matmul((codes, scales), (wc, np.zeros((2, 1), np.uint8)))
    with pytest.raises(ValueError, match="mismatch"):
        fp8.matmul((codes, scales), (np.zeros((32, 112), np.uint8), ws))
    with pytest.raises(ValueError, match="dtype"):
        fp8.matmul((codes, scales), (wc, ws), dtype=np.float64)
    with pytest.raises(ValueError, match="mismatch"):
        fp8.gated_gelu((codes, scales), (wc, ws), (wc, ws.astype(np.float32)))
    with pytest.raises(_lib.T5HError):
        fp8.quantize(np.zeros((2, 20), np.float32))
    assert fp8.scale_rows(1) == 16 and fp8.scale_rows(16) == 16 and fp8.scale_rows(17) == 32
