"""The linears of an encoder layer on 8-bit floating point (e4m3), on the GPU.

No counterpart in the reference, whose products are f32, bf16 or Q4_K x Q8_K.  Every block of 128
values along the summed axis has a scale.  Activations are coded in blocks of one row, with a power
of two as the scale: ``codes`` [M, K] u8 and ``scales`` [ceil(K/128), M16] u8 (the exponent's byte,
M16 = M rounded up to 16).  Weights are coded in blocks of 128 x 128: ``codes`` [N, K] u8 and
``scales`` [ceil(N/128), ceil(K/128)], bytes (E8M0) or f32 (F32_SCALES).
  * ``quantize(x)``             -- activations -> codes, scales
  * ``quantize_weights(w)``     -- weights -> codes, scales
  * ``rmsnorm(x, gamma, ...)``  -- residual's addition, T5LayerNorm (src/quantized_t5.rs:163-172), codes
  * ``matmul(a, w)``            -- A . W^T in f32, f16 or bf16
  * ``gated_gelu(a, w0, w1)``   -- gelu(A . W0^T) * (A . W1^T) (:231-249) as the next product's codes
The ``*_device`` forms take raw device addresses of the current device and enqueue on ``stream``;
bf16 buffers go through them.  Everything runs in libt5hip.so; there is no CPU fallback.  Shape and
type errors raise ValueError, what the library refuses raises T5HError.
"""
from __future__ import annotations

import numpy as np

from ._lib import T5H_SCALE_E8M0, T5H_SCALE_F32, T5H_TYPE_BF16, T5H_TYPE_F16, T5H_TYPE_F32, check, lib

F32, F16, BF16 = T5H_TYPE_F32, T5H_TYPE_F16, T5H_TYPE_BF16
E8M0, F32_SCALES = T5H_SCALE_E8M0, T5H_SCALE_F32
BLOCK = 128

_NUMPY = {F32: np.float32, F16: np.float16}


def scale_rows(m: int) -> int:
    """The row stride of activations' scales: m rounded up to 16."""
    return (m + 15) // 16 * 16


def _blocks(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


def _fits(bits: int) -> None:
    """`bits`, sizes and type codes or-ed together, is what the library's 32-bit arguments hold: ctypes
    would pass the low bits of a larger number."""
    if bits >> 31:
        raise ValueError("sizes and type codes must lie in 0 .. 2^31 - 1")


def _input(x: np.ndarray, name: str) -> tuple[np.ndarray, int]:
    x = np.ascontiguousarray(x)
    if x.ndim != 2:
        raise ValueError(f"{name} must be 2-D, got shape {x.shape}")
    for code, t in _NUMPY.items():
        if x.dtype == t:
            return x, code
    raise ValueError(f"{name} must be float32 or float16, got {x.dtype}")


def _activations(a) -> tuple[np.ndarray, np.ndarray]:
    codes, scales = a
    codes, scales = np.ascontiguousarray(codes), np.ascontiguousarray(scales)
    if codes.ndim != 2 or codes.dtype != np.uint8 or scales.dtype != np.uint8:
        raise ValueError("activations are a pair of uint8 arrays, codes [M, K] and scales")
    want = (_blocks(codes.shape[1]), scale_rows(codes.shape[0]))
    if scales.shape != want:
        raise ValueError(f"activation scales are {scales.shape}, codes {codes.shape} need {want}")
    return codes, scales


def _weights(w) -> tuple[np.ndarray, np.ndarray, int]:
    codes, scales = w
    codes, scales = np.ascontiguousarray(codes), np.ascontiguousarray(scales)
    if codes.ndim != 2 or codes.dtype != np.uint8 or scales.dtype not in (np.uint8, np.float32):
        raise ValueError("weights are a pair of arrays, codes [N, K] uint8 and scales uint8 or float32")
    want = (_blocks(codes.shape[0]), _blocks(codes.shape[1]))
    if scales.shape != want:
        raise ValueError(f"weight scales are {scales.shape}, codes {codes.shape} need {want}")
    return codes, scales, E8M0 if scales.dtype == np.uint8 else F32_SCALES


def quantize(x: np.ndarray, hip_device: int = 0) -> tuple[np.ndarray, np.ndarray]:
    """f32 or f16 activations [M, K] -> (codes [M, K], scales [ceil(K/128), M16])."""
    x, t = _input(x, "x")
    m, k = x.shape
    _fits(m | k)
    codes, scales = np.empty((m, k), np.uint8), np.zeros((_blocks(k), scale_rows(m)), np.uint8)
    check(lib.t5h_fp8_quantize(hip_device, x.ctypes.data, t, m, k, codes.ctypes.data, scales.ctypes.data))
    return codes, scales


def quantize_weights(w: np.ndarray, scale_type: int = E8M0, hip_device: int = 0) -> tuple[np.ndarray, np.ndarray]:
    """f32 or f16 weights [N, K] -> (codes [N, K], scales [ceil(N/128), ceil(K/128)])."""
    w, t = _input(w, "w")
    n, k = w.shape
    _fits(n | k | scale_type)
    codes = np.empty((n, k), np.uint8)
    scales = np.empty((_blocks(n), _blocks(k)), np.float32 if scale_type == F32_SCALES else np.uint8)
    check(lib.t5h_fp8_quantize_weights(hip_device, w.ctypes.data, t, n, k, scale_type, codes.ctypes.data,
                                       scales.ctypes.data))
    return codes, scales


def rmsnorm(x: np.ndarray, gamma: np.ndarray, eps: float = 1e-6, delta: np.ndarray | None = None,
            hip_device: int = 0):
    """T5LayerNorm of x + delta as codes: -> (codes, scales), and with a delta (codes, scales, sum),
    where sum is x + delta in x's type."""
    x, xt = _input(x, "x")
    m, d = x.shape
    _fits(m | d)
    gamma = np.ascontiguousarray(gamma, np.float32)
    if gamma.shape != (d,):
        raise ValueError(f"gamma is {gamma.shape}, rows have {d} values")
    codes, scales = np.empty((m, d), np.uint8), np.zeros((_blocks(d), scale_rows(m)), np.uint8)
    dp, dt, total = None, F32, None
    if delta is not None:
        delta, dt = _input(delta, "delta")
        if delta.shape != x.shape:
            raise ValueError(f"delta is {delta.shape}, x {x.shape}")
        dp, total = delta.ctypes.data, np.empty_like(x)
    check(lib.t5h_fp8_rmsnorm(hip_device, x.ctypes.data, xt, dp, dt, m, d, gamma.ctypes.data, eps,
                              None if total is None else total.ctypes.data, codes.ctypes.data, scales.ctypes.data))
    return (codes, scales) if total is None else (codes, scales, total)


def matmul(a, w, dtype=np.float32, hip_device: int = 0) -> np.ndarray:
    """A . W^T of activations a = (codes, scales) and weights w = (codes, scales): [M, N] f32 or f16."""
    ac, asc = _activations(a)
    wc, wsc, st = _weights(w)
    (m, k), (n, k2) = ac.shape, wc.shape
    _fits(m | n | k)
    if k != k2:
        raise ValueError(f"matmul dimension mismatch: a is [{m},{k}], w is [{n},{k2}]")
    types = [c for c, t in _NUMPY.items() if np.dtype(t) == np.dtype(dtype)]
    if not types:
        raise ValueError(f"dtype must be float32 or float16, got {dtype}")
    c = np.empty((m, n), dtype)
    check(lib.t5h_fp8_matmul(hip_device, ac.ctypes.data, asc.ctypes.data, m, wc.ctypes.data, wsc.ctypes.data, n, k, st,
                             c.ctypes.data, types[0]))
    return c


def gated_gelu(a, w0, w1, hip_device: int = 0) -> tuple[np.ndarray, np.ndarray]:
    """gelu(A . W0^T) * (A . W1^T) as activations (codes [M, N], scales [ceil(N/128), M16])."""
    ac, asc = _activations(a)
    c0, s0, st = _weights(w0)
    c1, s1, st1 = _weights(w1)
    (m, k), (n, k2) = ac.shape, c0.shape
    _fits(m | n | k)
    if k != k2 or c1.shape != c0.shape or st1 != st:
        raise ValueError(f"gated_gelu mismatch: a is [{m},{k}], w0 {c0.shape} {s0.dtype}, w1 {c1.shape} {s1.dtype}")
    codes, scales = np.empty((m, n), np.uint8), np.zeros((_blocks(n), scale_rows(m)), np.uint8)
    check(lib.t5h_fp8_gated_gelu(hip_device, ac.ctypes.data, asc.ctypes.data, m, c0.ctypes.data, s0.ctypes.data,
                                 c1.ctypes.data, s1.ctypes.data, n, k, st, codes.ctypes.data, scales.ctypes.data))
    return codes, scales


def quantize_device(d_x: int, type: int, m: int, k: int, d_codes: int, d_scales: int, stream: int = 0) -> None:
    """Activations of `type` (F32, F16, BF16) -> codes and scales, asynchronous on `stream`."""
    _fits(type | m | k)
    check(lib.t5h_fp8_quantize_device(d_x, type, m, k, d_codes, d_scales, stream))


def quantize_weights_device(d_w: int, type: int, n: int, k: int, scale_type: int, d_codes: int, d_scales: int,
                            stream: int = 0) -> None:
    """Weights of `type` -> codes and scales of `scale_type` (E8M0, F32_SCALES), on `stream`."""
    _fits(type | n | k | scale_type)
    check(lib.t5h_fp8_quantize_weights_device(d_w, type, n, k, scale_type, d_codes, d_scales, stream))


def rmsnorm_device(d_x: int, x_type: int, d_delta: int, delta_type: int, m: int, d: int, d_gamma: int, eps: float,
                   d_sum: int, d_codes: int, d_scales: int, stream: int = 0) -> None:
    """Residual's addition, T5LayerNorm and codes on `stream`; d_delta and d_sum may be 0 (none), and
    d_sum may be d_x."""
    _fits(x_type | delta_type | m | d)
    check(lib.t5h_fp8_rmsnorm_device(d_x, x_type, d_delta, delta_type, m, d, d_gamma, eps, d_sum, d_codes, d_scales,
                                     stream))


def matmul_device(d_a: int, d_a_scales: int, m: int, d_w: int, d_w_scales: int, n: int, k: int, scale_type: int,
                  d_c: int, c_type: int, stream: int = 0) -> None:
    """C [m, n] of `c_type` = A . W^T on `stream`."""
    _fits(m | n | k | scale_type | c_type)
    check(lib.t5h_fp8_matmul_device(d_a, d_a_scales, m, d_w, d_w_scales, n, k, scale_type, d_c, c_type, stream))


def gated_gelu_device(d_a: int, d_a_scales: int, m: int, d_w0: int, d_w0_scales: int, d_w1: int, d_w1_scales: int,
                      n: int, k: int, scale_type: int, d_codes: int, d_scales: int, stream: int = 0) -> None:
    """gelu(A . W0^T) * (A . W1^T) -> codes [m, n] and scales on `stream`."""
    _fits(m | n | k | scale_type)
    check(lib.t5h_fp8_gated_gelu_device(d_a, d_a_scales, m, d_w0, d_w0_scales, d_w1, d_w1_scales, n, k, scale_type,
                                        d_codes, d_scales, stream))
