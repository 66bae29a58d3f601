"""Sizes past what the kernels index are refused before anything is launched."""
import ctypes

import pytest

import candle_moe as cm

P = ctypes.c_void_p(4096)  # never read


@pytest.mark.parametrize("H", [2 ** 31 - 256, 2 ** 31 - 1])
@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_norm_refuses_rows_whose_last_step_passes_32_bits(H, dtype):
    rc = cm.lib().candle_moe_add_rms_norm(P, None, P, None, P, None, None, 1, H, 1e-6, dtype, None)
    assert rc == cm.CANDLE_MOE_ERR_INVALID and "hidden_dim must be in" in cm.last_error()
