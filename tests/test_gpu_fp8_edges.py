"""The 8-bit operators where values, types and places meet their limits.

The definition's own arithmetic is exact in every case below, so results are compared bit for bit: powers
of two, small integers, and sums of two values rounded once.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_fp8 import (E8M0, EPS, F32S, NORM_REL, TABLE, TYPES, _blocks, _byte_of, _check_codes, _gated, _guarded, _matmul,
                          _operand, _round_e4m3, _rows16, _same_codes, _stream, _unit_scales, _untouched, DEV, fp8)  # noqa: E402, F401


# ---- the norm's sum in the place of a delta of the other 16-bit type ---------------------------

@pytest.mark.parametrize("D", [16, 768, 1040, 2048, 4112, 16384, 16400])
@pytest.mark.parametrize("xk,dk", [("f16", "bf16"), ("bf16", "f16")])
def test_rmsnorm_sum_over_another_type(fp8, xk, dk, D):
    """x's type replaces the delta's bits in its own buffer; rows past 16,384 are read a second time, from there."""
    (xc, xt), (dc, dt), M = TYPES[xk], TYPES[dk], 7
    g = torch.Generator(device=DEV).manual_seed(D)
    x = torch.randn(M, D, generator=g, device=DEV).to(xt)
    delta = (0.5 * torch.randn(M, D, generator=g, device=DEV)).to(dt)
    gamma = 1 + 0.3 * torch.randn(D, generator=g, device=DEV)
    h = (x.float() + delta.float()).to(xt)
    raw, codes = _guarded(M * D)
    sraw, scales = _guarded(_blocks(D) * _rows16(M))
    place, total = _guarded(M * D, xt)
    total.view(dt).copy_(delta.view(-1))
    before = x.clone()
    fp8.rmsnorm_device(x.data_ptr(), xc, total.data_ptr(), dc, M, D, gamma.data_ptr(), 1e-6, total.data_ptr(),
                       codes.data_ptr(), scales.data_ptr(), _stream())
    torch.cuda.synchronize()
    assert _untouched(raw, codes) and _untouched(sraw, scales) and _untouched(place, total)
    assert torch.equal(x.view(torch.uint8), before.view(torch.uint8))
    assert torch.equal(total.view(M, D).view(torch.uint8), h.view(torch.uint8))
    h = h.double().cpu().numpy()
    y = h / np.sqrt((h * h).mean(1, keepdims=True) + 1e-6) * gamma.double().cpu().numpy()
    _check_codes(codes.cpu().numpy().reshape(M, D), scales.cpu().numpy().reshape(_blocks(D), -1)[:, :M], y, NORM_REL)


# ---- values below 2^-126 ----------------------------------------------------------------------

def _tiny(n):
    """e4m3 values times 2^-126 in turn: subnormal f32 below 1, down to 2^-135 and its ties."""
    v = np.array([2.0 ** -9, 3 * 2.0 ** -10, 2.0 ** -4, 0.1875, 0.5, 0.75, 1.0, 1.75, 0.0, -0.5, -0.875])
    return np.resize(v, n)


def test_quantizers_keep_subnormal_values(fp8):
    M, K = 20, 144
    want = np.stack([_tiny(K + i)[i:] for i in range(M)])
    x = torch.from_numpy(want * 2.0 ** -126).float().to(DEV)
    assert np.array_equal(x.double().cpu().numpy() * 2.0 ** 126, want)
    codes, scales = torch.empty(M, K, dtype=torch.uint8, device=DEV), torch.zeros(2, 32, dtype=torch.uint8, device=DEV)
    fp8.quantize_device(x.data_ptr(), 0, M, K, codes.data_ptr(), scales.data_ptr(), _stream())
    assert bool((scales[:, :M] == 1).all()) and _same_codes(codes.cpu().numpy(), _round_e4m3(want))
    for st, t in ((E8M0, torch.uint8), (F32S, torch.float32)):
        blocks = torch.empty(1, 2, dtype=t, device=DEV)
        fp8.quantize_weights_device(x.data_ptr(), 0, M, K, st, codes.data_ptr(), blocks.data_ptr(), _stream())
        assert bool((blocks == (1 if st == E8M0 else 2.0 ** -126)).all())
        assert _same_codes(codes.cpu().numpy(), _round_e4m3(want))


@pytest.mark.parametrize("M,N", [(1, 144), (70, 272), (700, 1424), (1100, 1040), (2100, 1040), (4200, 1040)])
def test_gated_keeps_subnormal_values(fp8, M, N):
    """gelu(2^-63) = 2^-64 to 2^-63 of it; times 2^-62 v it is v 2^-126: every strip's codes, exactly."""
    K = 144
    a, w0, w1 = np.zeros((M, K)), np.zeros((N, K)), np.zeros((N, K))
    a[:, 3], a[:, 130] = 1, 1
    w0[:, 3], w1[:, 130] = 1, np.where(np.arange(N) % 11 == 1, 0.0, _tiny(N))
    byte = np.stack([np.full(M, 127 - 63), np.full(M, 127 - 62)])
    ac, asc = _operand(a, byte, M, K)
    w = [torch.from_numpy(_round_e4m3(v)).to(DEV) for v in (w0, w1)]
    unit = _unit_scales(N, K, False)
    codes, s = _gated(fp8, ac, asc, w[0], unit, w[1], unit, E8M0)
    assert (s == 1).all()
    assert _same_codes(codes, np.broadcast_to(_round_e4m3(w1[:, 130]), (M, N)))
