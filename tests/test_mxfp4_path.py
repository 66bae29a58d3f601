"""fused_moe_mxfp4_path / _kernel: what they answer for sizes (no GPU needed)."""
import pytest

import candle_moe as cm


@pytest.fixture
def policies():
    yield
    cm.set_tile_policy(cm.TILE_AUTO)
    cm.set_combine_policy(cm.COMBINE_AUTO)


def test_invalid_sizes():
    assert cm.fused_moe_mxfp4_path(4, 96, 80, 4, 2, 1) == cm.PATH_NAMES[-1]
    assert cm.fused_moe_mxfp4_kernel(4, 64, 96, 4, 2, 2) == -1  # f32
    assert cm.fused_moe_mxfp4_kernel(4, 64, 96, 0, 2, 1) == -1


def test_decode_and_prefill():
    assert cm.fused_moe_mxfp4_kernel(1, 2048, 768, 128, 8, 1) == cm.TILE_DEC_GEMV
    assert cm.fused_moe_mxfp4_path(1, 2048, 768, 128, 8, 1) == "pairs"
    assert cm.fused_moe_mxfp4_kernel(16384, 4096, 1536, 8, 2, 1, 0, True) == cm.TILE_W8
    assert cm.fused_moe_mxfp4_path(16384, 4096, 1536, 8, 2, 1, 0, True) == "expert-set"
    assert cm.fused_moe_mxfp4_path(4096, 2048, 768, 128, 8, 1) == "pairs"


def test_policies(policies):
    cm.set_combine_policy(cm.COMBINE_EXPERT_SETS)
    for tile in (cm.TILE_LDS_128, cm.TILE_W8, cm.TILE_128x256_OCC2, cm.TILE_ROWS32):
        cm.set_tile_policy(tile)
        assert cm.fused_moe_mxfp4_kernel(300, 256, 256, 3, 2, 1) == tile
        # (32-row tiles have no expert sets; K tiles of up to 128 end with an expert)
        assert cm.fused_moe_mxfp4_path(300, 256, 256, 3, 2, 1) == ("pairs" if tile == cm.TILE_ROWS32 else "expert-set")
        assert cm.fused_moe_mxfp4_path(300, 256, 192, 3, 2, 1) == "pairs"
