"""Every kernel of the MoE over MXFP4 weights on the sizes where tiles end: K of
whole and half K tiles, scale rows that start at any byte, groups around the tile
heights and their extensions, both combine paths, K splits."""
import pytest
import torch

import candle_moe as cm
import operator_reference as ref
from test_gpu_mxfp4 import BF, F16, check, run, setup, want

pytestmark = pytest.mark.gpu
TILES = [cm.TILE_LDS_128, cm.TILE_W8, cm.TILE_ROWS32, cm.TILE_128x256_OCC2, cm.TILE_DEC_GEMV]


@pytest.fixture
def policies():
    yield
    cm.set_tile_policy(cm.TILE_AUTO)
    cm.set_combine_policy(cm.COMBINE_AUTO)


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("moe_type", [0, 1])
@pytest.mark.parametrize("T, H, I, E, k", [(1, 32, 32, 1, 1), (3, 96, 160, 2, 1), (65, 416, 288, 3, 2), (129, 288, 352, 2, 1),
                                          (160, 64, 96, 1, 1), (161, 736, 224, 1, 1), (257, 320, 544, 2, 2), (300, 1056, 96, 5, 3)])
def test_each_kernel(T, H, I, E, k, moe_type, tile, policies):
    cm.set_tile_policy(tile)
    check(setup(T, H, I, E, k, moe_type, BF if T % 2 else F16, T % 3 == 0, seed=T), T % 3)


@pytest.mark.parametrize("tile", [cm.TILE_LDS_128, cm.TILE_W8, cm.TILE_128x256_OCC2])
@pytest.mark.parametrize("moe_type", [0, 1])
@pytest.mark.parametrize("T, H, I, E, k", [(40, 96, 64, 3, 2), (161, 288, 192, 2, 2), (700, 544, 128, 4, 1)])
def test_expert_sets(T, H, I, E, k, moe_type, tile, policies):
    cm.set_tile_policy(tile)
    cm.set_combine_policy(cm.COMBINE_EXPERT_SETS)
    s = setup(T, H, I, E, k, moe_type, BF, False, seed=T, dropped=0.1)
    # (the routing weight goes into the intermediate before its rounding: the
    # same bound, without the pair row's)
    check(s, 0)
    out = torch.ones(T, H, dtype=BF, device="cuda")
    y, far = want(s, 0)
    run(s, 0, out, accumulate=True)
    ref.within(out, y + 1, far + 2.0 ** -8 * ((y + 1).abs() + far))


@pytest.mark.parametrize("tile", [cm.TILE_LDS_128, cm.TILE_W8, cm.TILE_ROWS32, cm.TILE_128x256_OCC2])
def test_long_k_in_splits(tile, policies):
    # few tiles over a long K: the 32-row kernel's splits, the 256x256 kernel's tail
    cm.set_tile_policy(tile)
    check(setup(33, 4128, 2080, 2, 1, 0, BF, False, seed=4), 0)
    check(setup(300, 2080, 4128, 2, 1, 1, BF, False, seed=5), 1)


@pytest.mark.parametrize("sets", [False, True])
@pytest.mark.parametrize("moe_type", [0, 1])
@pytest.mark.parametrize("T, H, I, E, k", [(1, 128, 32, 1, 1), (130, 256, 160, 2, 2), (257, 384, 288, 1, 1), (300, 128, 544, 5, 3),
                                          (600, 1152, 256, 2, 1), (700, 4224, 128, 4, 2)])
def test_eight_bit_rows_as_they_are(T, H, I, E, k, moe_type, sets, policies):
    # the gate/up and fc1 products in the MX formats themselves (256x256 tiles)
    cm.set_tile_policy(cm.TILE_W8)
    cm.set_combine_policy(cm.COMBINE_EXPERT_SETS if sets else cm.COMBINE_PAIRS)
    s = setup(T, H, I, E, k, moe_type, BF, True, seed=T, dropped=0.1)
    first = check(s, T % 3, aligned=2.0 ** -12)
    assert torch.equal(first, check(s, T % 3, aligned=2.0 ** -12))


def test_eight_bit_rows_with_scales_far_apart(policies):
    cm.set_tile_policy(cm.TILE_W8)
    s = setup(40, 512, 128, 2, 1, 0, BF, True, seed=11)
    for q in (s["x_scale"], s["gate"][1], s["up"][1]):
        q.copy_((120 + (torch.arange(q.numel(), device="cuda") * 7) % 11).to(torch.uint8).view_as(q))
    s["x_scale"][3] = 0
    check(s, 2, aligned=2.0 ** -12)
    s["gate"][1][1, 5] = 255
    hit = (s["idx"] == 1).any(1)
    # (SiLU: the ReLU, max(x, 0), takes a NaN to 0 as everywhere here)
    out = run(s, 0, torch.empty(40, 512, dtype=BF, device="cuda"))
    assert torch.isnan(out[hit]).all() and not torch.isnan(out[~hit]).any()


@pytest.mark.parametrize("tile", TILES)
def test_foreign_scales_do_not_reach_the_columns_of_an_expert(tile, policies):
    # K = 3 * 32: the half tile past the end of a row lies before the next row's
    # scales; a NaN there belongs to that row alone
    cm.set_tile_policy(tile)
    s = setup(40, 96, 96, 2, 1, 1, BF, False, seed=7)
    s["up"][1][:, 5, :] = 255  # fc2's output column 5
    out = run(s, 1, torch.zeros(40, 96, dtype=BF, device="cuda"))
    nan = torch.isnan(out)
    assert nan[:, 5].all() and not nan[:, :5].any() and not nan[:, 6:].any()


@pytest.mark.parametrize("tile", TILES)
def test_same_bits_every_time(tile, policies):
    cm.set_tile_policy(tile)
    s = setup(90, 1024, 512, 8, 2, 0, BF, False, seed=8)
    first = run(s, 0, torch.empty(90, 1024, dtype=BF, device="cuda"))
    for _ in range(5):
        assert torch.equal(first, run(s, 0, torch.empty_like(first)))


def test_an_unaligned_view_of_the_scales_is_refused(policies):
    s = setup(4, 64, 64, 2, 1, 0, BF, False)
    flat = torch.zeros(s["gate"][1].numel() + 1, dtype=torch.uint8, device="cuda")
    s["gate"] = (s["gate"][0], flat[1:].view_as(s["gate"][1]))
    with pytest.raises(cm.CandleMoeError, match="scales must be 16-byte aligned"):
        run(s, 0, torch.empty(4, 64, dtype=BF, device="cuda"))
