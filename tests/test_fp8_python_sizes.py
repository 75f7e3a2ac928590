"""Sizes that a 32-bit argument does not hold are refused, not cut to their low bits (no GPU needed)."""
import pytest

from witchcraft_amd import fp8

P = 1 << 20          # an aligned address, which nothing reads
WRAPS = 1 << 32      # 0 in 32 bits: with it every call below would find nothing to do, and succeed


@pytest.mark.parametrize("size", [WRAPS, -WRAPS, 1 << 31, -1])
def test_device_forms_refuse_sizes(size):
    for call in (lambda: fp8.quantize_device(P, fp8.F32, size, 128, P, P),
                 lambda: fp8.quantize_device(P, fp8.F32, 0, WRAPS + 128, P, P),
                 lambda: fp8.quantize_device(P, WRAPS, 0, 128, P, P),
                 lambda: fp8.quantize_weights_device(P, fp8.F32, size, 128, fp8.E8M0, P, P),
                 lambda: fp8.quantize_weights_device(P, fp8.F32, 0, 128, WRAPS, P, P),
                 lambda: fp8.rmsnorm_device(P, fp8.F32, 0, 0, size, 128, P, 1e-6, 0, P, P),
                 lambda: fp8.rmsnorm_device(P, fp8.F32, P, WRAPS, 0, 128, P, 1e-6, 0, P, P),
                 lambda: fp8.matmul_device(P, P, size, P, P, 16, 128, fp8.E8M0, P, fp8.F32),
                 lambda: fp8.matmul_device(P, P, 16, P, P, size, 128, fp8.E8M0, P, fp8.F32),
                 lambda: fp8.matmul_device(P, P, 0, P, P, 16, WRAPS + 128, fp8.E8M0, P, fp8.F32),
                 lambda: fp8.gated_gelu_device(P, P, size, P, P, P, P, 16, 128, fp8.E8M0, P, P),
                 lambda: fp8.gated_gelu_device(P, P, 16, P, P, P, P, size, 128, fp8.E8M0, P, P)):
        with pytest.raises(ValueError, match="2\\^31"):
            call()


def test_scale_type_of_weights():
    import numpy as np
    with pytest.raises(ValueError, match="2\\^31"):
        fp8.quantize_weights(np.zeros((0, 128), np.float32), scale_type=WRAPS)
