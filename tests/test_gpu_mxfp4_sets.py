"""MXFP4 down / fc2 over expert sets: the change of the experts' codes and scales along
K, on every tile that has the path, both dtypes, writing and accumulating."""
import pytest
import torch

import candle_moe as cm
import operator_reference as ref
from test_gpu_mxfp4 import BF, F16, run, setup

pytestmark = pytest.mark.gpu
CODE = {F16: 0, BF: 1}


@pytest.fixture
def policies():
    yield
    cm.set_tile_policy(cm.TILE_AUTO)
    cm.set_combine_policy(cm.COMBINE_AUTO)


def want(s, act, sets, aligned=0.0):
    """In 64 bits, and how far a result may be: no rounding of a pair's row. Over sets
    the f32 sum runs over k I terms in place of I (at most (k - 1) I 2^-24 of what the
    intermediate's rounding u leaves, per u), and the weight goes into the intermediate
    before its rounding (the least step's half by itself, not times the weight)."""
    x = s["x"] if s["x_scale"] is None else ref.from_mxfp8(s["x"], s["x_scale"])
    w = [ref.from_mxfp4(*q) if q[0] is not None else None for q in (s["gate"], s["up"], s["down"])]
    dtype, E, k = s["dtype"], s["E"], s["k"]
    y, far = ref.moe(x, *w, s["rw"], s["idx"], act, s["moe_type"], dtype, rounded=False, aligned=aligned)
    if sets:
        last = w[2] if w[2] is not None else w[1]
        mags = torch.cat((last.abs().sum(-1), torch.zeros_like(last[:1, :, 0])))  # (a dropped pair: nothing)
        idx = torch.where((s["idx"] < 0) | (s["idx"] >= E), E, s["idx"]).long()
        far = far * (1 + (k - 1) * last.shape[2] * 2.0 ** -24 / ref.HALF[dtype]) + ref.LEAST[dtype] * mags[idx].sum(1)
    return y, far


def check_both(s, act, sets, aligned=0.0):
    T, H = s["x"].shape
    dtype = s["dtype"]
    y, far = want(s, act, sets, aligned)
    out = run(s, act, torch.full((T, H), float("nan"), dtype=dtype, device="cuda"))
    ref.within(out, y, far, "written")
    assert torch.equal(out, run(s, act, torch.empty_like(out)))
    acc = torch.randn(T, H, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
    total = y + acc.double()
    run(s, act, acc, accumulate=True)
    ref.within(acc, total, far + ref.HALF[dtype] * (total.abs() + far), "accumulated")


@pytest.mark.parametrize("tile", [cm.TILE_LDS_128, cm.TILE_W8, cm.TILE_128x256_OCC2])
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("moe_type", [0, 1])
@pytest.mark.parametrize("T, H, I, E, k", [(40, 96, 128, 3, 2), (161, 288, 256, 2, 2), (150, 160, 384, 3, 3), (700, 544, 128, 4, 2),
                                           (400, 96, 384, 2, 2), (289, 320, 256, 4, 3)])
def test_sets(T, H, I, E, k, moe_type, dtype, tile, policies):
    cm.set_tile_policy(tile)
    cm.set_combine_policy(cm.COMBINE_EXPERT_SETS)
    assert cm.fused_moe_mxfp4_path(T, H, I, E, k, CODE[dtype], moe_type) == "expert-set"
    check_both(setup(T, H, I, E, k, moe_type, dtype, False, seed=T, dropped=0.1), T % 3, True)
    check_both(setup(T, H, I, E, k, moe_type, dtype, False, seed=T + 1), T % 3, True)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("T, H, I, E, k", [(300, 256, 256, 3, 2), (290, 384, 384, 3, 3)])
def test_sets_from_8_bit_rows(T, H, I, E, k, dtype, policies):
    for tile in (cm.TILE_LDS_128, cm.TILE_W8, cm.TILE_128x256_OCC2):
        cm.set_tile_policy(tile)
        cm.set_combine_policy(cm.COMBINE_EXPERT_SETS)
        assert cm.fused_moe_mxfp4_path(T, H, I, E, k, CODE[dtype], 0, True) == "expert-set"
        check_both(setup(T, H, I, E, k, 0, dtype, True, seed=T), 0, True, aligned=2.0 ** -12)


@pytest.mark.parametrize("tile", [cm.TILE_LDS_128, cm.TILE_W8, cm.TILE_128x256_OCC2, cm.TILE_ROWS32])
@pytest.mark.parametrize("T, H, I, E, k", [(40, 96, 64, 3, 2), (161, 288, 192, 2, 2)])
def test_other_intermediate_sizes_take_pairs(T, H, I, E, k, tile, policies):
    cm.set_tile_policy(tile)
    cm.set_combine_policy(cm.COMBINE_EXPERT_SETS)
    assert cm.fused_moe_mxfp4_path(T, H, I, E, k, 1) == "pairs"
    check_both(setup(T, H, I, E, k, 0, BF, False, seed=T, dropped=0.1), 1, False)


@pytest.mark.parametrize("tile", [cm.TILE_DEC_GEMV, cm.TILE_ROWS32, cm.TILE_LDS_128, cm.TILE_128x256_OCC2, cm.TILE_W8])
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("moe_type", [0, 1])
@pytest.mark.parametrize("T, H, I, E, k", [(1, 256, 128, 8, 2), (5, 2048, 768, 16, 4), (33, 416, 288, 8, 2), (130, 288, 96, 5, 3),
                                           (300, 512, 256, 4, 2)])
def test_pair_rows_are_not_rounded(T, H, I, E, k, moe_type, dtype, tile, policies):
    cm.set_tile_policy(tile)
    cm.set_combine_policy(cm.COMBINE_PAIRS)
    check_both(setup(T, H, I, E, k, moe_type, dtype, False, seed=T + 3, dropped=0.05), T % 3, False)
