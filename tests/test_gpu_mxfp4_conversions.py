"""The MoE's own conversions of MXFP4 weights and MXFP8 rows: every code at every scale
that the dtype holds, on every kernel, bit for bit (products with one term)."""
import pytest
import torch

import candle_moe as cm
import operator_reference as ref

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16
N = 4096
TILES = [cm.TILE_DEC_GEMV, cm.TILE_ROWS32, cm.TILE_LDS_128, cm.TILE_128x256_OCC2, cm.TILE_W8]


@pytest.fixture
def policies():
    yield
    cm.set_tile_policy(cm.TILE_AUTO)


def pack(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def one_per_row(code, at):
    """Codes [1, N, N / 2] with `code` [N] at k = at [N], zeros elsewhere; scales of 2^0."""
    c = torch.zeros((N, N), dtype=torch.uint8, device="cuda")
    c[torch.arange(N, device="cuda"), at] = code
    return pack(c)[None].contiguous(), torch.full((1, N, N // 32), 127, dtype=torch.uint8, device="cuda")


def run(x, gate, up, down, dtype, moe_type, x_scale=None):
    T = x.shape[0]
    out = torch.full((T, N), 7.0, dtype=dtype, device="cuda")
    cm.fused_moe_mxfp4(x, gate[0], up[0], down[0], gate[1], up[1], down[1], torch.ones(T, 1, device="cuda"),
                       torch.zeros(T, 1, dtype=torch.int32, device="cuda"), out, 1, 1, activation=2, moe_type=moe_type,
                       input_scale=x_scale, accumulate=False)
    return out


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("rows8", [False, True])
def test_weights(dtype, rows8, tile, policies):
    cm.set_tile_policy(tile)
    n = torch.arange(N, device="cuda")
    scale, code = n // 16, n % 16
    codes = (code | (code << 4)).to(torch.uint8).view(N, 1).expand(N, 16).contiguous()
    value = ref.from_mxfp4(codes, scale.to(torch.uint8).view(N, 1))[:, 0]
    # (what the dtype does not hold, infinite or a NaN, would reach every output)
    held = torch.isfinite(value) & (value.abs() <= torch.finfo(dtype).max)
    value = torch.where(held, value, 0.0)
    at = n * 37 % N
    up = one_per_row(torch.where(held, code, 0).to(torch.uint8), at)
    up[1][0, n, at // 32] = torch.where(held, scale, 127).to(torch.uint8)
    ones = lambda k: one_per_row(torch.full((N,), 2, dtype=torch.uint8, device="cuda"), k)  # noqa: E731
    if rows8:
        x = torch.full((2, N), 0x38, dtype=torch.uint8, device="cuda")
        s = torch.full((2, N // 32), 127, dtype=torch.uint8, device="cuda")
    else:
        x, s = torch.ones(2, N, dtype=dtype, device="cuda"), None
    out = run(x, ones(n * 0 + 5), up, ones(n), dtype, 0, s)
    want = value.float().to(dtype)
    for t in range(2):
        bad = out[t] != want
        assert not bad.any(), [(int(scale[i]), int(code[i]), float(out[t, i]), float(want[i])) for i in bad.nonzero()[:4, 0]]


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("dtype", [BF, F16])
def test_rows(dtype, tile, policies):
    cm.set_tile_policy(tile)
    # token t: 16 scales, each with its 256 codes
    code = torch.arange(N, device="cuda") % 256
    scale = torch.arange(16, device="cuda").view(16, 1) * 16 + torch.arange(N // 32, device="cuda") // 8
    code = code.expand(16, N).to(torch.uint8).contiguous()
    value = ref.from_mxfp8(code, scale.to(torch.uint8).contiguous())
    held = torch.isfinite(value) & (value.abs() <= torch.finfo(dtype).max)
    value = torch.where(held, value, 0.0)
    x = torch.where(held, code, 0).to(torch.uint8)
    s = torch.where(scale == 255, 127, scale).to(torch.uint8).contiguous()
    n = torch.arange(N, device="cuda")
    last = one_per_row(torch.full((N,), 2, dtype=torch.uint8, device="cuda"), n)
    for sign, c in ((1.0, 2), (-1.0, 10)):  # (the ReLU takes one sign at a time)
        first = one_per_row(torch.full((N,), c, dtype=torch.uint8, device="cuda"), n)
        out = run(x, first, last, (None, None), dtype, 1, s)
        want = (sign * value).float().to(dtype).clamp_min(0)
        bad = out != want
        assert not bad.any(), [(int(s[t, i // 32]), int(x[t, i]), float(out[t, i]), float(want[t, i]))
                               for t, i in bad.nonzero()[:4].tolist()]
