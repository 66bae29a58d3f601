"""add_rms_norm against its definition in 64 bits. The f32 arithmetic before the
one rounding: a sum of squares over chains of at most 128 fused steps and 16 joins
(144 * 2^-24 of the sum, half of that after the root), z's own rounding and four
more: below 80 * 2^-24 < 2^-17 of a value."""
import pytest
import torch

import candle_moe as cm
import operator_reference as ref

pytestmark = pytest.mark.gpu
F32 = 2.0 ** -17
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def inputs(T, H, dtype, seed=1, residual=True):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, H, generator=g) * torch.exp2(torch.randn(T, 1, generator=g))).to(dtype).cuda()
    r = (torch.randn(T, H, generator=g) * 2).to(dtype).cuda() if residual else None
    return x, r, (1 + 0.1 * torch.randn(H, generator=g)).to(dtype).cuda()


def check_mx(codes, scales, y):
    """Within half a step of e4m3 at that scale (2^-4 of the value, 2^-10 * 2^e
    below the normal range), the scale the least that holds the block."""
    most = y.unflatten(-1, (-1, 32)).abs().amax(-1)
    lo, hi = ref.mx_scale(most * (1 - F32), 448.0), ref.mx_scale(most * (1 + F32), 448.0)
    assert ((scales == lo) | (scales == hi)).all()
    unit = ref.scale_value(scales).repeat_interleave(32, -1)
    far = torch.maximum(y.abs() * 2.0 ** -4, unit * 2.0 ** -10) + F32 * y.abs()
    ref.within(ref.from_mxfp8(codes, scales), y, far, "MXFP8")
    assert ref.from_mxfp8(codes, scales).abs().max() <= 448 * unit.max()


def check(x, r, w, eps=1e-6, mx=True):
    T, H = x.shape
    z, y = ref.norm(x, w, eps, r)
    u, tiny = ref.HALF[x.dtype], ref.LEAST[x.dtype]
    out, ro = torch.full_like(x, 7), torch.full_like(x, 7)
    codes = torch.full((T, H), 7, dtype=torch.uint8, device="cuda") if mx else None
    scales = torch.full((T, H // 32), 7, dtype=torch.uint8, device="cuda") if mx else None
    cm.add_rms_norm(x, w, eps, residual=r, residual_output=ro, output=out, codes=codes, scales=scales)
    ref.within(ro, z, u * z.abs() * (1 + F32) + 2.0 ** -24 * z.abs() + tiny, "residual")
    ref.within(out, y, u * y.abs() * (1 + F32) + F32 * y.abs() + tiny, "output")
    if mx:
        check_mx(codes, scales, y)
    return out, ro, codes, scales


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T, H", [(1, 32), (5, 64), (3, 512), (67, 544), (2, 1024), (9, 1056), (1, 2048), (33, 2880),
                                  (4, 4096), (3, 4128), (2, 8192), (2, 8224), (1, 32768), (1000, 256)])
def test_with_and_without_a_residual(T, H, dtype):
    for residual in (True, False):
        check(*inputs(T, H, dtype, T + H, residual))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T, H", [(3, 1), (5, 7), (2, 100), (4, 1001), (1, 40000), (7, 8), (3, 1000)])
def test_sizes_without_an_8_bit_form(T, H, dtype):
    check(*inputs(T, H, dtype, T + H), mx=False)


@pytest.mark.parametrize("dtype", DTYPES)
def test_each_output_alone_and_in_place(dtype):
    x, r, w = inputs(19, 736, dtype)
    out, ro, codes, scales = check(x, r, w)
    o2 = torch.empty_like(x)
    cm.add_rms_norm(x, w, 1e-6, residual=r, output=o2)
    assert torch.equal(o2, out)
    c2, s2 = torch.empty_like(codes), torch.empty_like(scales)
    cm.add_rms_norm(x, w, 1e-6, residual=r, codes=c2, scales=s2)
    assert torch.equal(c2, codes) and torch.equal(s2, scales)
    x2, r2 = x.clone(), r.clone()
    cm.add_rms_norm(x2, w, 1e-6, residual=r2, residual_output=r2, output=x2)
    assert torch.equal(x2, out) and torch.equal(r2, ro)
    # one element off alignment: the general kernel, the same within its rounding
    H = 736
    flat = [torch.empty(t.numel() + 1, dtype=dtype, device="cuda")[1:].view_as(t) for t in (x, r)]
    for f, t in zip(flat, (x, r)):
        f.copy_(t)
    cm.add_rms_norm(flat[0], w, 1e-6, residual=flat[1], residual_output=flat[1], output=flat[0])
    assert torch.equal(flat[1], ro)
    y = ref.norm(x, w, 1e-6, r)[1]
    ref.within(flat[0], y, ref.HALF[dtype] * y.abs() * (1 + F32) + F32 * y.abs() + ref.LEAST[dtype])


def test_blocks_of_zeros_and_borders_of_the_scale():
    # rows whose norm is 1 to the last bit: y = x (eps 0, mean of squares 1)
    x = torch.zeros(4, 64, device="cuda")
    x[0, :32] = 1.0
    x[0, :16] *= 2 ** 0.5
    x[1, 40] = 8.0          # 32 zeros before it
    x[2] = 1.0
    x[3, ::2] = 2 ** 0.5
    w = torch.ones(64, device="cuda")
    _, _, codes, scales = check(x, None, w, eps=0.0)
    assert scales[1, 0] == 0 and (codes[1, :32] == 0).all()
    # 1 = 256 * 2^-8 (448 * 2^-9 < 1 <= 448 * 2^-8)
    assert (scales[2] == 119).all() and (codes[2] == codes[2, 0]).all()
    # amax just at, just above 448 * 2^e by the weight
    for amax, e in ((448.0, 0), (448.0 + 2.0 ** -15, 1), (449.0, 1), (3.5, -7), (3.5 * (1 + 2.0 ** -23), -6)):
        w = torch.full((64,), amax, device="cuda")
        c, s = torch.empty(1, 64, dtype=torch.uint8, device="cuda"), torch.empty(1, 2, dtype=torch.uint8, device="cuda")
        cm.add_rms_norm(torch.ones(1, 64, device="cuda"), w, 0.0, codes=c, scales=s)
        assert (s == 127 + e).all()


def test_what_is_not_finite_stays_in_its_row():
    x, r, w = inputs(4, 64, torch.float32)
    x[1, 5], x[2, 40] = float("nan"), float("inf")
    out = torch.empty_like(x)
    c, s = torch.empty(4, 64, dtype=torch.uint8, device="cuda"), torch.empty(4, 2, dtype=torch.uint8, device="cuda")
    cm.add_rms_norm(x, w, 1e-6, residual=r, output=out, codes=c, scales=s)
    y = ref.norm(x, w, 1e-6, r)[1]
    assert torch.equal(torch.isnan(out), torch.isnan(y))
    assert (s[1] == 255).all() and s[2, 1] == 255 and s[2, 0] == 0
    assert ((c[1] & 127) == 127).all()
    ref.within(out[[0, 3]], y[[0, 3]], F32 * 2 * y[[0, 3]].abs())
    # a row of zeros: 0 with eps, NaN without (0 / 0)
    z = torch.zeros(1, 64, device="cuda")
    cm.add_rms_norm(z, w, 1e-6, output=out[:1], codes=c[:1], scales=s[:1])
    assert (out[0] == 0).all() and (s[0] == 0).all() and (c[0] == 0).all()
    cm.add_rms_norm(z, w, 0.0, output=out[:1])
    assert torch.isnan(out[0]).all()


def test_rows_past_the_batch_and_a_graph():
    x, r, w = inputs(6, 2048, torch.bfloat16)
    out, ro = torch.full_like(x, 3), torch.full_like(x, 3)
    c = torch.full((6, 2048), 3, dtype=torch.uint8, device="cuda")
    s = torch.full((6, 64), 3, dtype=torch.uint8, device="cuda")
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        cm.add_rms_norm(x[:5], w, 1e-6, residual=r[:5], residual_output=ro[:5], output=out[:5], codes=c[:5], scales=s[:5])
    for seed in (5, 6, 7):
        x.copy_(inputs(6, 2048, torch.bfloat16, seed)[0])
        g.replay()
        torch.cuda.synchronize()
        want = check(x[:5], r[:5], w)
        for got, b in zip((out, ro, c, s), want):
            assert torch.equal(got[:5], b) and (got[5] == 3).all()
