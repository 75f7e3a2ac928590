"""Queries and keys between the projection and attention, on the GPU: head norms and rotation by positions.

No counterpart in the reference, whose attention has a bias by distance instead.  In one pass every
head of q and k is normed (x / sqrt(mean x^2 + eps) * gamma) and its first ``rot`` values are turned, in
pairs, by position * frequency.  Positions are int32 and may have several axes (row and column; time,
height and width); each pair follows one of them.
  * ``frequencies(rot, theta)``      -- theta^(-2i / rot), the usual ladder, f64
  * ``table(freqs, axes)``           -- a pair's frequency and axis as the GPU takes them, u64
  * ``rotate(q, k, positions, ...)`` -- numpy arrays in f32 or f16
  * ``rotate_device(...)``           -- raw device addresses of the current device, on ``stream``; rows may
    lie apart, so q and k can be columns of one projection's rows
Everything runs in libt5hip.so; there is no CPU fallback.  Shape and type errors raise ValueError, what the
library refuses raises T5HError.
"""
from __future__ import annotations

import numpy as np

from ._lib import (T5H_ROTARY_HALVES, T5H_ROTARY_NEIGHBOURS, T5H_TYPE_BF16, T5H_TYPE_F16, T5H_TYPE_F32, check, lib)

F32, F16, BF16 = T5H_TYPE_F32, T5H_TYPE_F16, T5H_TYPE_BF16
HALVES, NEIGHBOURS = T5H_ROTARY_HALVES, T5H_ROTARY_NEIGHBOURS

_NUMPY = {F32: np.float32, F16: np.float16}


def _fits(bits: int, strides: int = 0) -> None:
    """`bits`, sizes and codes or-ed together, and `strides` are what the library's 32- and 64-bit arguments
    hold: ctypes would pass the low bits of a larger number."""
    if bits >> 31 or strides >> 63:
        raise ValueError("sizes and codes must lie in 0 .. 2^31 - 1, strides in 0 .. 2^63 - 1")


def frequencies(rot: int, theta: float = 10000.0) -> np.ndarray:
    """theta^(-2i / rot) for the rot / 2 pairs, in radians per step."""
    return float(theta) ** (-np.arange(0, rot, 2, dtype=np.float64) / rot)


def table(freqs, axes=None) -> np.ndarray:
    """The table of pairs' frequencies (radians per step) and axes (0 .. 7; None: all 0).  Angles are within 2^-27 of
    position * frequency; each turn (2 pi) a step past the first adds up to 2^-28 at positions of 2^31."""
    freqs = np.ascontiguousarray(freqs, np.float64)
    if freqs.ndim != 1:
        raise ValueError(f"frequencies must be 1-D, got shape {freqs.shape}")
    _fits(freqs.size)
    if axes is not None:
        given = np.asarray(axes)
        if given.shape != freqs.shape or not np.issubdtype(given.dtype, np.integer) and given.size:
            raise ValueError(f"axes must be whole numbers, one per frequency, got {given.dtype} {given.shape}")
        if given.size and (given.min() < 0 or given.max() > 7):
            raise ValueError("axes must lie in 0 .. 7")
        axes = np.ascontiguousarray(given, np.int32)
    out = np.empty(freqs.shape, np.uint64)
    check(lib.t5h_rotary_table(freqs.ctypes.data, None if axes is None else axes.ctypes.data, freqs.size, out.ctypes.data))
    return out


def _heads(x: np.ndarray, name: str) -> tuple[np.ndarray, int]:
    x = np.ascontiguousarray(x)
    if x.ndim != 3:
        raise ValueError(f"{name} must be [rows, heads, values], got shape {x.shape}")
    for code, t in _NUMPY.items():
        if x.dtype == t:
            return x, code
    raise ValueError(f"{name} must be float32 or float16, got {x.dtype}")


def _gamma(gamma, d: int, name: str):
    if gamma is None:
        return None
    gamma = np.ascontiguousarray(gamma, np.float32)
    if gamma.shape != (d,):
        raise ValueError(f"{name} is {gamma.shape}, heads have {d} values")
    return gamma


def rotate(q: np.ndarray, k: np.ndarray, positions, table: np.ndarray, q_gamma=None, k_gamma=None, eps: float = 1e-6,
           pairing: int = HALVES, hip_device: int = 0) -> tuple[np.ndarray, np.ndarray]:
    """q [T, Hq, D] and k [T, Hk, D] normed (where there is a gamma [D]) and turned by positions [T] or [axes, T];
    the table's pairs are the first values of each head."""
    q, t = _heads(q, "q")
    k, kt = _heads(k, "k")
    if kt != t or k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2]:
        raise ValueError(f"q is {q.dtype} {q.shape}, k {k.dtype} {k.shape}")
    rows, qh, d = q.shape
    given = np.asarray(positions)
    given = given[None] if given.ndim == 1 else given
    if given.ndim != 2 or given.shape[1] != rows or not np.issubdtype(given.dtype, np.integer) and given.size:
        raise ValueError(f"positions must be whole numbers [T] or [axes, T], got {given.dtype} {given.shape}")
    if given.size and (given.min() < -2 ** 31 or given.max() >= 2 ** 31):
        raise ValueError("positions must fit 32 bits")
    pos = np.ascontiguousarray(given, np.int32)
    tab = np.ascontiguousarray(table)
    if tab.ndim != 1 or tab.dtype != np.uint64:
        raise ValueError("the table is what table() returns")
    qg, kg = _gamma(q_gamma, d, "q_gamma"), _gamma(k_gamma, d, "k_gamma")
    _fits(rows | qh | k.shape[1] | d | 2 * tab.size | pos.shape[0] | pairing)
    q_out, k_out = np.empty_like(q), np.empty_like(k)
    check(lib.t5h_rotary(hip_device, q.ctypes.data, qh, k.ctypes.data, k.shape[1], t, rows, d,
                         None if qg is None else qg.ctypes.data, None if kg is None else kg.ctypes.data, eps,
                         tab.ctypes.data, 2 * tab.size, pairing, pos.ctypes.data, pos.shape[0], q_out.ctypes.data,
                         k_out.ctypes.data))
    return q_out, k_out


def rotate_device(d_q: int, ldq: int, q_heads: int, d_k: int, ldk: int, k_heads: int, type: int, t: int, d: int,
                  d_q_gamma: int, d_k_gamma: int, eps: float, d_table: int, rot: int, pairing: int, d_pos: int,
                  axes: int, d_q_out: int, ldq_out: int, d_k_out: int, ldk_out: int, stream: int = 0) -> None:
    """Head norms and rotation of t rows on `stream`; ld*: values from row to row.  Gammas may be 0 (no norm),
    outputs the inputs themselves."""
    _fits(q_heads | k_heads | type | t | d | rot | pairing | axes, ldq | ldk | ldq_out | ldk_out)
    check(lib.t5h_rotary_device(d_q, ldq, q_heads, d_k, ldk, k_heads, type, t, d, d_q_gamma, d_k_gamma, eps, d_table, rot,
                                pairing, d_pos, axes, d_q_out, ldq_out, d_k_out, ldk_out, stream))
