"""Low-rank adapters of many requests at once beside a shared projection, on the GPU.

No counterpart in the reference, whose encoder has one set of weights.  Each row of a packed batch has the
adapter ``ids[t]`` or none (an id outside 0 .. G - 1), and y = x W^T, which ``fp8.matmul`` or any other product
computed for all rows alike, becomes y + scale * (x A^T) B^T.  ``a`` [G, slices, R, K], ``b`` [G, N, R]; a slice
is a part of y's columns with an A of its own, as q, k and v of a fused projection are.
  * ``add(x, ids, a, b, y, ...)``  -- numpy arrays; x in f16, or codes and scales as ``fp8`` returns them
  * ``add_device(...)``            -- raw device addresses of the current device, on ``stream``
  * ``workspace_bytes(...)``       -- the device memory that ``add_device`` needs beside them
Everything runs in libt5hip.so; there is no CPU fallback.  Shape and type errors raise ValueError, what the
library refuses raises T5HError.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from ._lib import T5H_TYPE_BF16, T5H_TYPE_E4M3, T5H_TYPE_F16, T5H_TYPE_F32, check, lib

F32, F16, BF16, E4M3 = T5H_TYPE_F32, T5H_TYPE_F16, T5H_TYPE_BF16, T5H_TYPE_E4M3


def _fits(bits: int, wide: int = 0) -> None:
    """`bits`, sizes and codes or-ed together, and `wide`, row lengths and bytes, are what the library's 32- and
    64-bit arguments hold: ctypes would pass the low bits of a larger number."""
    if bits >> 31 or wide >> 63:
        raise ValueError("sizes and codes must lie in 0 .. 2^31 - 1, strides and bytes in 0 .. 2^63 - 1")


def _columns(cols):
    for n in cols:
        _fits(n)
    return (C.c_int32 * len(cols))(*cols)


def workspace_bytes(t: int, k: int, slices: int, rank: int) -> int:
    """Bytes of device memory for add_device with these sizes."""
    _fits(t | k | slices | rank)
    out = C.c_size_t()
    check(lib.t5h_adapter_workspace(t, k, slices, rank, C.byref(out)))
    return out.value


def add(x, ids, a: np.ndarray, b: np.ndarray, y: np.ndarray, scales=None, ranks=None, cols=None,
        hip_device: int = 0) -> np.ndarray:
    """y [T, N] (f32 or f16) + scales[ids] * (x a[ids]^T) b[ids]^T: x [T, K] f16 or (codes, scales); a, b f16; ranks: whole
    numbers [G], how many of each adapter's R count (None: all; outside 0 .. R the nearer of both), where b is finite up to
    the next multiple of 8; cols: the slices' columns (None: all alike)."""
    if isinstance(x, tuple):
        codes, xs = (np.ascontiguousarray(v) for v in x)
        if codes.ndim != 2 or codes.dtype != np.uint8 or xs.dtype != np.uint8:
            raise ValueError("activations are a pair of uint8 arrays, codes [T, K] and scales")
        want = ((codes.shape[1] + 127) // 128, (codes.shape[0] + 15) // 16 * 16)
        if xs.shape != want:
            raise ValueError(f"activation scales are {xs.shape}, codes {codes.shape} need {want}")
        rows, xt = codes, E4M3
    else:
        rows, xs, xt = np.ascontiguousarray(x), None, F16
        if rows.ndim != 2 or rows.dtype != np.float16:
            raise ValueError(f"x must be [T, K] float16, or codes and scales, got {rows.dtype} {rows.shape}")
    t, k = rows.shape
    a, b, y = np.ascontiguousarray(a), np.ascontiguousarray(b), np.ascontiguousarray(y)
    if a.dtype != np.float16 or b.dtype != np.float16 or a.ndim != 4 or b.ndim != 3:
        raise ValueError("a [G, slices, R, K] and b [G, N, R] must be float16")
    g, slices, r = a.shape[:3]
    if a.shape[3] != k or b.shape[0] != g or b.shape[2] != r:
        raise ValueError(f"x has rows of {k} values, a is {a.shape}, b {b.shape}")
    if y.dtype not in (np.float32, np.float16) or y.shape != (t, b.shape[1]):
        raise ValueError(f"y must be [{t}, {b.shape[1]}] float32 or float16, got {y.dtype} {y.shape}")
    if cols is None:
        if slices == 0 or b.shape[1] % slices:
            raise ValueError(f"{b.shape[1]} columns are not {slices} slices")
        cols = (b.shape[1] // slices,) * slices
    if len(cols) != slices or sum(cols) != b.shape[1]:
        raise ValueError(f"slices of {tuple(cols)} columns, a has {slices}, b {b.shape[1]} columns")
    given = np.asarray(ids)
    if given.shape != (t,) or not np.issubdtype(given.dtype, np.integer) and given.size:
        raise ValueError(f"ids must be whole numbers, one for each of {t} rows, got {given.dtype} {given.shape}")
    which = np.ascontiguousarray(np.where((given < 0) | (given >= g), -1, given), np.int32)
    sp = None if scales is None else np.ascontiguousarray(scales, np.float32)
    own = None if ranks is None else np.asarray(ranks)
    if own is not None and not np.issubdtype(own.dtype, np.integer) and own.size:
        raise ValueError(f"ranks must be whole numbers, got {own.dtype} {own.shape}")
    rp = None if own is None else np.ascontiguousarray(np.where(own < 0, 0, np.where(own > r, r, own)), np.int32)
    for name, v in (("scales", sp), ("ranks", rp)):
        if v is not None and v.shape != (g,):
            raise ValueError(f"{name} are {v.shape}, there are {g} adapters")
    _fits(t | k | g | r | slices)
    out = np.empty_like(y)
    columns = _columns(cols)
    check(lib.t5h_adapter_add(hip_device, rows.ctypes.data, xt, None if xs is None else xs.ctypes.data, t, k,
                              which.ctypes.data, g, a.ctypes.data, b.ctypes.data, F16, None if rp is None else rp.ctypes.data,
                              None if sp is None else sp.ctypes.data, r, C.addressof(columns), slices, y.ctypes.data,
                              out.ctypes.data, F32 if y.dtype == np.float32 else F16))
    return out


def add_device(d_x: int, x_type: int, d_x_scales: int, ldx: int, t: int, k: int, d_ids: int, adapters: int, d_a: int,
               d_b: int, w_type: int, d_ranks: int, d_scales: int, rank: int, cols, d_y: int, ldy: int, d_out: int, ldo: int,
               y_type: int, d_work: int, work_bytes: int, stream: int = 0) -> None:
    """out = y + what the adapters add, on `stream`.  cols: the slices' columns; d_x_scales (rows of f16 or bf16),
    d_ranks (all of `rank`) and d_scales (all 1) may be 0; d_out may be d_y."""
    _fits(x_type | t | k | adapters | w_type | rank | y_type, ldx | ldy | ldo | work_bytes)
    columns = _columns(cols)
    check(lib.t5h_adapter_add_device(d_x, x_type, d_x_scales, ldx, t, k, d_ids, adapters, d_a, d_b, w_type, d_ranks, d_scales,
                                     rank, C.addressof(columns), len(cols), d_y, ldy, d_out, ldo, y_type, d_work, work_bytes,
                                     stream))
