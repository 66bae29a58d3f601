"""add_rms_norm on rows near the ends of f32's range, and how near its results are to
64 bits: the norm is good to 2^-40, so an output is off by its dtype's rounding
(after one to f32), 8-bit codes and scales are those of the exact y."""
import pytest
import torch

import candle_moe as cm
import operator_reference as ref
from test_gpu_rms_norm import DTYPES, inputs

pytestmark = pytest.mark.gpu
ONCE = 2.0 ** -24 + 2.0 ** -38  # y to f32 (2^-24 of it), from a value within 2^-40 and two products


def outputs(x, w, eps, r=None, mx=True):
    T, H = x.shape
    out = torch.full_like(x, 7)
    codes = torch.full((T, H), 7, dtype=torch.uint8, device="cuda") if mx else None
    scales = torch.full((T, H // 32), 7, dtype=torch.uint8, device="cuda") if mx else None
    cm.add_rms_norm(x, w, eps, residual=r, output=out, codes=codes, scales=scales)
    return out, codes, scales


def check(x, w, eps, r=None, mx=True):
    z = x if r is None else (x.float() + r.float())  # (z is an f32 sum)
    y = ref.norm(z, w, float(torch.tensor(eps, dtype=torch.float32)))[1]  # (eps is an f32)
    out, codes, scales = outputs(x, w, eps, r, mx)
    u = ref.HALF[x.dtype] if x.dtype != torch.float32 else 0.0
    ref.within(out, y, y.abs() * (ONCE + u * (1 + ONCE)) + ref.LEAST[x.dtype] + 2.0 ** -149, "output")
    if mx:
        b = y.unflatten(-1, (-1, 32))
        s = ref.mx_scale(b.abs().amax(-1), 448.0)
        assert torch.equal(scales, s)
        v = (b / ref.scale_value(s).unsqueeze(-1)).flatten(-2)
        # e4m3 of the exact value: steps of 2^-3 of the binade, of 2^-9 below 2^-6
        step = torch.exp2(torch.frexp(v).exponent.clamp_min(-5).double() - 4)
        assert torch.equal(codes.view(torch.float8_e4m3fn).float().double(), torch.round(v / step) * step)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T, H", [(3, 64), (5, 1024), (40, 2048), (33, 2880), (2, 16384)])
def test_as_near_as_promised(T, H, dtype):
    x, r, w = inputs(T, H, dtype, T + H)
    check(x, w, 1e-6, r)
    check(x, w, 1e-6)


@pytest.mark.parametrize("T, H", [(3, 7), (4, 1001), (1, 40000)])
def test_as_near_at_any_size(T, H):
    x, r, w = inputs(T, H, torch.float32, T + H)
    check(x, w, 1e-6, r, mx=False)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H", [64, 1056, 4096])
@pytest.mark.parametrize("e", [-148, -140, -133, -127, -120, -100, -60, 100, 108, 115, 120, 124, 126])
def test_rows_at_the_ends_of_the_range(e, H, dtype):
    # values around 2^e; in the smallest few steps of the type are left of them
    g = torch.Generator().manual_seed(H)
    x = (torch.randn(6, H, generator=g).clamp(-3, 3).double() * 2.0 ** e).to(dtype).cuda()
    x[:, ::5] = (2.0 ** e if e > -133 or dtype == torch.float32 else 2.0 ** -133)  # (no row of zeros)
    w = (1 + 0.1 * torch.randn(H, generator=g)).to(dtype).cuda()
    check(x, w, 0.0)
    check(x, w, 1e-6, mx=e >= -100)  # (below, y = 1000 x leaves the normal range of f32)
    flat = torch.empty(x.numel() + 1, dtype=dtype, device="cuda")[1:].view_as(x)  # the general kernel
    flat.copy_(x)
    check(flat, w, 0.0, mx=False)


def test_a_few_large_values_among_small_ones():
    x = torch.full((2, 512), 2.0 ** -120, device="cuda")
    x[0, 17], x[1, 400] = 3e38, -2.0 ** 127
    check(x, torch.ones(512, device="cuda"), 0.0, mx=False)
    x = torch.full((2, 512), 2.0 ** -149, device="cuda")
    x[0, 17] = 2.0 ** -126
    check(x, torch.ones(512, device="cuda"), 0.0)
