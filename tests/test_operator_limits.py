"""Sizes of topk_route past one launch and past 32-bit pair numbers are refused
before anything is launched."""
import ctypes

import pytest

import candle_moe as cm

P = ctypes.c_void_p(4096)  # never read


@pytest.mark.parametrize("T, E, k", [((1 << 25) + 1, 8, 1), (1 << 25, 64, 64), (2 ** 31 - 1, 1, 1)])
def test_route_refuses_what_one_launch_does_not_hold(T, E, k):
    rc = cm.lib().candle_moe_topk_route(P, 2, None, P, P, P, E, T, k, 0, 1, 1, 1, 1, 1.0, None)
    assert rc == cm.CANDLE_MOE_ERR_INVALID and "at most" in cm.last_error()
