"""The 8-bit products' limits on the largest activations, refused before any device work (no GPU needed).

Rows' scales are read through a buffer descriptor of ceil(K / 128) * M16 bytes, M16 = M rounded up to 16,
and lanes without a row read past its end, at 2^31 - 1: the scales have to end there.
"""
import numpy as np
import pytest

from witchcraft_amd import _lib

P = 1 << 20                # an aligned address, which nothing reads
M, K = 715827882, 272      # 3 M = 2^31 - 2 blocks, whose scales are 3 M16 = 2^31 + 16 bytes


def _refused(rc):
    msg = _lib.lib.t5h_last_error().decode()
    assert rc == _lib.T5H_ERR_INVALID and "scales" in msg, (rc, msg)


@pytest.mark.parametrize("m,k", [(M, K), ((1 << 30) - 15, 256), ((1 << 17) - 7, 1 << 21)])
def test_products_refuse_scales_past_2_31(m, k):
    blocks, m16 = -(-k // 128), -(-m // 16) * 16
    assert m * blocks < 1 << 31 <= m16 * blocks
    lib, buf = _lib.lib, np.zeros(64, np.uint8).ctypes.data
    _refused(lib.t5h_fp8_matmul_device(P, P, m, P, P, 16, k, 0, P, 0, None))
    _refused(lib.t5h_fp8_gated_gelu_device(P, P, m, P, P, P, P, 16, k, 0, P, P, None))
    _refused(lib.t5h_fp8_matmul(0, buf, buf, m, buf, buf, 16, k, 0, buf, 0))
    _refused(lib.t5h_fp8_gated_gelu(0, buf, buf, m, buf, buf, buf, buf, 16, k, 0, buf, buf))
