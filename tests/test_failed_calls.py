"""A call that fails leaves nothing behind: the next valid call on the thread succeeds.

HIP keeps a thread's last error until it is asked for, whatever succeeds in between, and a launch is
checked by asking.  A failed allocation that left its error there made the next call report it,
after its kernel had been enqueued and before its results were copied.
"""
import numpy as np
import pytest

from witchcraft_amd import _lib, codec, fp8, score

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


# Sizes whose buffers no card holds (half a TB and more), so that nothing is read from `buf`.
HUGE = (1 << 24) - 16, 16384


def _codes():
    x = np.full((3, 128), 448.0, np.float32)
    codes, scales = fp8.quantize(x)
    assert (codes == 0x7e).all() and (scales[0, :3] == 127).all()


def test_failed_allocation_leaves_no_error():
    m, k = HUGE
    buf = np.zeros(4096, np.uint8).ctypes.data
    lib = _lib.lib
    _codes()
    for call in (lambda: lib.t5h_fp8_quantize(0, buf, 0, m, k, buf, buf),
                 lambda: lib.t5h_fp8_quantize_weights(0, buf, 0, m, k, 0, buf, buf),
                 lambda: lib.t5h_fp8_rmsnorm(0, buf, 0, buf, 0, m, k, buf, 1e-6, buf, buf, buf),
                 lambda: lib.t5h_fp8_matmul(0, buf, buf, m, buf, buf, m, k, 0, buf, 0),
                 lambda: lib.t5h_fp8_gated_gelu(0, buf, buf, m, buf, buf, buf, buf, k, k, 0, buf, buf)):
        assert call() == _lib.T5H_ERR_NOMEM
        _codes()
        assert int(torch.ones(5, device="cuda:0").sum()) == 5


def test_failed_device_leaves_no_error():
    x = np.ones((3, 128), np.float32)
    with pytest.raises(_lib.T5HError):
        fp8.quantize(x, hip_device=4096)
    _codes()
    with pytest.raises(_lib.T5HError):
        codec.residual_to_q4_bytes(x, x, np.zeros(3, np.int32), hip_device=4096)
    _codes()
    with pytest.raises(_lib.T5HError):
        score.matmul_t(x, x, hip_device=4096)
    _codes()
