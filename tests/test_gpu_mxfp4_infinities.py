"""An intermediate that leaves the dtype's range is an infinity, and the products over
it are infinite too (no weight is zero): on every kernel and split of K, in its own
token alone."""
import pytest
import torch

import candle_moe as cm
import operator_reference as ref

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16


@pytest.fixture
def policies():
    yield
    cm.set_tile_policy(cm.TILE_AUTO)


@pytest.mark.parametrize("tile", [cm.TILE_AUTO, cm.TILE_DEC_GEMV, cm.TILE_ROWS32, cm.TILE_LDS_128, cm.TILE_128x256_OCC2,
                                  cm.TILE_W8])
@pytest.mark.parametrize("moe_type", [0, 1])
@pytest.mark.parametrize("dtype, big", [(F16, 2.0 ** 15), (BF, 2.0 ** 125)])
@pytest.mark.parametrize("T, H, I, E, k", [(2, 64, 96, 4, 1), (3, 96, 1056, 8, 2), (2, 64, 32, 8, 3), (2, 128, 160, 8, 5),
                                           (2, 64, 2048, 16, 8), (4, 64, 1280, 32, 16)])
def test_infinite_intermediates(T, H, I, E, k, moe_type, dtype, big, tile, policies):
    cm.set_tile_policy(tile)
    one = lambda n, m: (torch.full((E, n, m // 2), 0x22, dtype=torch.uint8, device="cuda"),  # noqa: E731
                        torch.full((E, n, m // 32), 127, dtype=torch.uint8, device="cuda"))
    # gate and up / fc1: 2^-10 (bf16 2^-100) everywhere but in column 3, 1 there
    gate = one(I, H)
    up = one(I, H) if moe_type == 0 else one(H, I)
    for q in (gate, up) if moe_type == 0 else (gate,):
        q[1].fill_(117 if dtype == F16 else 27)
        q[1][:, 3] = 127
    down = one(H, I) if moe_type == 0 else (None, None)
    x = torch.full((T, H), 2.0 ** -6, dtype=dtype, device="cuda")
    # column 3 of row 1: big by gate times big by up, or 8 big by fc1 alone
    x[1] = big / H * (8 if moe_type == 1 else 1)
    rw = torch.full((T, k), 1.0 / k, device="cuda")
    idx = torch.stack([torch.randperm(E, generator=torch.Generator().manual_seed(t))[:k] for t in range(T)]).int().cuda()
    out = torch.full((T, H), 7.0, dtype=dtype, device="cuda")
    cm.fused_moe_mxfp4(x, gate[0], up[0], down[0], gate[1], up[1], down[1], rw, idx, out, E, k, activation=2,
                       moe_type=moe_type, accumulate=False)
    assert (out[1] == float("inf")).all()
    rest = [t for t in range(T) if t != 1]
    w = [ref.from_mxfp4(*q) if q[0] is not None else None for q in (gate, up, down)]
    y, far = ref.moe(x[rest], *w, rw[rest], idx[rest], 2, moe_type, dtype, rounded=False)
    ref.within(out[rest], y, far)
