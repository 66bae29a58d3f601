"""The operators around the expert products where their launches take other
forms: every lane layout of topk_route's batches, batches past one launch of
add_rms_norm, decode batches of many pairs, repeated experts, rows in several K
chunks, 8-bit rows and scales that start anywhere, the binding against ctypes, and
all of it in one graph."""
import numpy as np
import pytest
import torch

import candle_moe as cm
import operator_reference as ref
from test_gpu_mxfp4 import BF, F16, check as check_moe, randn, run, setup, want
from test_gpu_topk_route import bias_of, call, check as check_route, logits_of

pytestmark = pytest.mark.gpu


# -------------------------------------------------------------------- topk_route
# (E, groups, chosen groups, group_top, k): from 2048 rows on 16 lanes of 4, 8 and
# 16 experts, 32 of 8 and 16, 64 of 8 and 16, the exact form (k of 63 on);
# experts a multiple of the lane's and not
LAYOUTS = [(64, 1, 1, 1, 14), (61, 1, 1, 1, 8), (128, 1, 1, 1, 8), (100, 1, 1, 1, 3), (256, 1, 1, 1, 8),
           (250, 1, 1, 1, 14), (256, 1, 1, 1, 20), (512, 1, 1, 1, 30), (500, 1, 1, 1, 8), (512, 1, 1, 1, 40),
           (1024, 1, 1, 1, 8), (256, 8, 4, 2, 8), (160, 8, 3, 1, 6), (96, 3, 2, 2, 8), (64, 16, 4, 1, 8),
           (512, 8, 2, 2, 8), (320, 5, 2, 2, 9), (1024, 32, 4, 2, 8), (72, 1, 1, 1, 70)]


@pytest.mark.parametrize("E, G, tg, top, k", LAYOUTS)
def test_many_rows(E, G, tg, top, k):
    T = 2051  # (not a multiple of the rows of a workgroup)
    kw = dict(num_groups=G, topk_groups=tg, group_top=top)
    check_route(logits_of(T, E, seed=E + k), k, bias_of(E), score="sigmoid", scale=2.5, **kw)
    # bf16 logits: many equal ones in a row, each a tie that goes to the lower index
    l = logits_of(T, E, BF, seed=E + k + 1, std=0.25)
    l[5], l[6, ::2], l[7, E // 2] = 0.0, -float("inf"), float("nan")
    l[8], l[9, 0] = -float("inf"), float("inf")
    check_route(l, k, score="softmax", renormalize=E % 3 != 0, **kw)


@pytest.mark.parametrize("E, G, tg", [(128, 1, 1), (256, 8, 4)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_many_rows_of_near_ties(E, G, tg, score):
    T = 2048
    l = logits_of(T, E, seed=5)
    l[:, E // 2:] = torch.nextafter(l[:, : E // 2], torch.full((), 9.0, device="cuda"))
    kw = dict(score=score, num_groups=G, topk_groups=tg, group_top=1)
    check_route(l, 8, **kw)
    p = torch.sigmoid(l[0].double()) if score == "sigmoid" else torch.softmax(l[0].double(), 0)
    check_route(l, 8, (0.25 - p).float(), **kw)  # row 0: all c within an f32 rounding of 0.25
    check_route(l, 8, bias_of(E, std=1e6), **kw)  # a bias that leaves few bits for the scores


def test_past_one_launch_of_rows():
    T, H = (1 << 21) + 5, 32
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(T, H, device="cuda", generator=g, dtype=BF)
    w = torch.randn(H, device="cuda", generator=g, dtype=BF)
    y, r = torch.zeros_like(x), torch.zeros_like(x)
    codes, scales = (torch.zeros(T, n, dtype=torch.uint8, device="cuda") for n in (H, 1))
    cm.add_rms_norm(x, w, 1e-6, residual=x, residual_output=r, output=y, codes=codes, scales=scales)
    part = torch.cat((torch.arange(0, 9), torch.arange((1 << 21) - 9, T))).cuda()
    z, want_y = ref.norm(x[part], w, 1e-6, x[part])
    # the output's rounding and 2^-17 of f32 arithmetic; codes: half a step of 2^-3 of
    # the value, or of the least step, 2^-10 of the block's power of two
    ref.within(y[part], want_y, (2.0 ** -8 * (1 + 2.0 ** -8) + 2.0 ** -17) * want_y.abs())
    back = ref.from_mxfp8(codes[part], scales[part])
    least = ref.scale_value(scales[part]) * 2.0 ** -10
    ref.within(back, want_y, (2.0 ** -4 * (1 + 2.0 ** -4) + 2.0 ** -17) * want_y.abs() + least)
    assert torch.equal(r[part], (2 * x[part].float()).to(BF))


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("T, H", [(1500, 2048), (3000, 480), (40, 16384)])
def test_codes_are_those_of_the_exact_norm(T, H, dtype):
    # scales and codes of the 64-bit y itself, each rounded once: a y rounded to f32
    # on the way would change some 2 of these 3 million codes
    g = torch.Generator(device="cuda").manual_seed(T)
    x, r = (torch.randn(T, H, device="cuda", generator=g).to(dtype) for _ in range(2))
    w = (1 + 0.1 * torch.randn(H, device="cuda", generator=g)).to(dtype)
    codes, scales = (torch.empty(T, n, dtype=torch.uint8, device="cuda") for n in (H, H // 32))
    cm.add_rms_norm(x, w, 1e-6, residual=r, codes=codes, scales=scales)
    z = (x.float() + r.float()).double()  # (as the kernel's z)
    _, y = ref.norm(z, w, float(np.float32(1e-6)))
    b = y.unflatten(-1, (-1, 32))
    s = ref.mx_scale(b.abs().amax(-1), 448.0)
    assert torch.equal(scales, s)
    v = b / ref.scale_value(s).unsqueeze(-1)
    step = torch.exp2(torch.floor(torch.log2(v.abs())).clamp(min=-6) - 3)
    want_v = torch.round(v / step) * step
    assert torch.equal(codes.view(torch.float8_e4m3fn).double(), want_v.flatten(-2))


# ------------------------------------------------------------- decode of MXFP4
@pytest.mark.parametrize("rows8", [False, True])
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("T, H, I, E, k", [(32, 2080, 1536, 8, 2), (20, 4128, 96, 3, 3), (40, 352, 2080, 5, 3),
                                          (128, 160, 224, 100, 1), (17, 8192, 64, 2, 1), (8, 64, 8224, 2, 2),
                                          (1, 16384, 32, 4, 2)])
def test_decode_of_many_pairs_and_long_rows(T, H, I, E, k, dtype, rows8):
    # 17 to 128 rows of an expert (two row blocks, several rounds of them) in one or
    # more K chunks, K no multiple of a step
    for mt in (0, 1):
        s = setup(T, H, I, E, k, mt, dtype, rows8, seed=T + I)
        cm.set_tile_policy(cm.TILE_DEC_GEMV)
        try:
            check_moe(s, (T + mt) % 3)
        finally:
            cm.set_tile_policy(cm.TILE_AUTO)


@pytest.mark.parametrize("moe_type", [0, 1])
@pytest.mark.parametrize("T, H, I, E, k", [(1, 64, 96, 2, 1), (1, 256, 1536, 8, 2), (1, 32, 32, 40, 16), (2, 96, 160, 64, 9),
                                          (1, 128, 4096, 16, 3), (1, 64, 4128, 16, 3), (1, 64, 128, 40, 17), (1, 2048, 768, 128, 8),
                                          (3, 512, 1056, 100, 5), (9, 768, 2048, 8, 1), (12, 320, 736, 200, 10)])
def test_a_few_tokens_with_their_sums(T, H, I, E, k, moe_type):
    # 1 to 8 K parts of a slot, several slots of a wave, dropped pairs, both outputs
    dt = BF if T % 2 else F16
    s = setup(T, H, I, E, k, moe_type, dt, moe_type == 1, seed=T + I, dropped=0.0 if E == 2 else 0.2)
    first = check_moe(s, (T + k) % 3)
    assert torch.equal(first, check_moe(s, (T + k) % 3))
    big = randn(T + 1, H, seed=9).to(dt).cuda()
    before = big.clone()
    y, far = want(s, 0)
    run(s, 0, big[:T], accumulate=True)
    total = before[:T].double() + y
    ref.within(big[:T], total, far + ref.HALF[dt] * (total.abs() + far))
    assert torch.equal(big[T:], before[T:])
    s["idx"].fill_(E)
    assert (run(s, 0, torch.ones(T, H, dtype=dt, device="cuda")) == 0).all()


@pytest.mark.parametrize("tile", [cm.TILE_DEC_GEMV, cm.TILE_ROWS32, cm.TILE_LDS_128, cm.TILE_W8])
@pytest.mark.parametrize("rows8", [False, True])
def test_one_expert_in_every_slot(tile, rows8):
    # more rows of an expert than tokens
    cm.set_tile_policy(tile)
    try:
        for T, k in ((3, 8), (20, 4), (10, 12)):
            s = setup(T, 256, 128, 16, k, 0, BF, rows8, seed=T)
            s["idx"].fill_(7)
            s["idx"][1, 1] = 2
            check_moe(s, 0, aligned=2.0 ** -12 if rows8 and tile == cm.TILE_W8 else 0.0)
    finally:
        cm.set_tile_policy(cm.TILE_AUTO)


@pytest.mark.parametrize("tile", [cm.TILE_DEC_GEMV, cm.TILE_ROWS32, cm.TILE_W8])
@pytest.mark.parametrize("H", [96, 256, 1152])
def test_row_scales_that_start_anywhere(tile, H):
    cm.set_tile_policy(tile)
    try:
        s = setup(30, H, 64, 4, 2, 0, BF, True, seed=H)
        whole = run(s, 0, torch.empty(30, H, dtype=BF, device="cuda"))
        for at in (1, 2, 4):
            flat = torch.full((s["x_scale"].numel() + at,), 255, dtype=torch.uint8, device="cuda")
            flat[at:] = s["x_scale"].flatten()
            moved = dict(s, x_scale=flat[at:].view_as(s["x_scale"]))
            got = check_moe(moved, 0, aligned=2.0 ** -12 if tile == cm.TILE_W8 else 0.0)
            if tile != cm.TILE_W8 or at == 4:
                assert torch.equal(got, whole)
    finally:
        cm.set_tile_policy(cm.TILE_AUTO)


@pytest.mark.parametrize("T, H, I, E, k, rows8", [(280, 2048, 1536, 8, 2, False), (300, 2048, 768, 32, 4, True),
                                                 (700, 1280, 256, 16, 4, True), (2000, 256, 128, 8, 2, False)])
def test_automatic_choice_of_larger_batches(T, H, I, E, k, rows8):
    for mt in (0, 1):
        check_moe(setup(T, H, I, E, k, mt, BF, rows8, seed=T), mt, aligned=2.0 ** -12 if rows8 else 0.0)


# ------------------------------------------------- binding, streams and graphs
def test_the_binding_and_ctypes_give_the_same(monkeypatch):
    if cm._native is None:
        pytest.skip("candle_moe._fast is not built")

    def all_of_them():
        out = list(call(logits_of(9, 64), 4, bias_of(64), score="sigmoid", num_groups=4, topk_groups=2))
        x, w = randn(5, 256, seed=1).to(BF).cuda(), randn(256, seed=2).to(BF).cuda()
        y, r = torch.empty_like(x), torch.empty_like(x)
        c, s = (torch.empty(5, n, dtype=torch.uint8, device="cuda") for n in (256, 8))
        cm.add_rms_norm(x, w, 1e-5, residual=x, residual_output=r, output=y, codes=c, scales=s)
        out += [t.float().cpu().numpy() for t in (y, r, c, s)]
        for rows8 in (False, True):
            for mt in (0, 1):
                z = setup(5, 256, 128, 8, 2, mt, BF, rows8)
                o = randn(5, 256, seed=3).to(BF).cuda()
                out.append(run(z, mt, o, accumulate=not rows8).float().cpu().numpy())
        return out

    native = all_of_them()
    monkeypatch.setattr(cm, "_native", None)
    for a, b in zip(native, all_of_them()):
        assert np.array_equal(a, b)


def test_captures_of_smaller_batches_on_both_sides_of_the_decode_kernels():
    H, I, E, k = 2048, 1408, 8, 2  # (37 MB of codes and scales)
    s = setup(64, H, I, E, k, 0, BF, False, seed=2)
    cut = {T: dict(s, **{n: s[n][:T].contiguous() for n in ("x", "rw", "idx")}) for T in (64, 56, 49, 48, 40, 9)}
    outs = {T: torch.empty(T, H, dtype=BF, device="cuda") for T in cut}
    cm.trim_workspaces()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run(cut[64], 0, outs[64])
    torch.cuda.synchronize()
    graphs = {}
    for T in cut:
        graphs[T] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graphs[T], stream=side):
            run(cut[T], 0, outs[T])
    for T, g in graphs.items():
        eager = run(cut[T], 0, torch.empty_like(outs[T]))
        outs[T].zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(eager, outs[T]), T
    ref.within(outs[56], *want(cut[56], 0))


@pytest.mark.parametrize("T, H, I, E, k, tile", [(24, 512, 256, 16, 4, cm.TILE_AUTO), (300, 512, 256, 8, 2, cm.TILE_W8),
                                                (600, 256, 128, 4, 1, cm.TILE_128x256_OCC2)])
def test_a_block_in_one_graph(T, H, I, E, k, tile):
    """Norm, logits, routing and 8-bit rows through the experts, captured together and
    replayed on new inputs between eager calls on another stream."""
    w = (1 + 0.1 * randn(H, seed=3)).to(BF).cuda()
    router = randn(H, E, seed=4, std=0.05).cuda()
    mats = [cm.quantize_mxfp4(randn(E, a, b, seed=s, std=0.05).to(BF).cuda())
            for a, b, s in ((H, I, 6), (H, I, 7), (I, H, 8))]
    (g, gs), (u, us), (d, ds) = mats

    def buffers():
        e = lambda *s, dt=BF: torch.zeros(s, dtype=dt, device="cuda")  # noqa: E731
        return dict(x=e(T, H), r=e(T, H), y=e(T, H), c=e(T, H, dt=torch.uint8), s=e(T, H // 32, dt=torch.uint8),
                    rw=e(T, k, dt=torch.float32), i=e(T, k, dt=torch.int32), ei=e(T, k, dt=torch.int32))

    def block(b):
        cm.add_rms_norm(b["x"], w, 1e-6, residual=b["r"], residual_output=b["r"], output=b["y"], codes=b["c"], scales=b["s"])
        cm.topk_route(b["y"].float() @ router, b["rw"], b["i"], b["ei"], score="sigmoid")
        cm.fused_moe_mxfp4(b["c"], g, u, d, gs, us, ds, b["rw"], b["i"], b["r"], E, k, input_scale=b["s"])

    def fill(b, seed):
        b["x"].copy_(randn(T, H, seed=seed).to(BF))
        b["r"].copy_(randn(T, H, seed=seed + 1).to(BF))

    cm.set_tile_policy(tile)
    try:
        caught, eager, side, other = buffers(), buffers(), torch.cuda.Stream(), torch.cuda.Stream()
        with torch.cuda.stream(side):
            fill(caught, 20)
            block(caught)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            block(caught)
        for seed in (30, 40, 50):
            fill(caught, seed)
            fill(eager, seed)
            torch.cuda.synchronize()
            # (the graph uses the workspace of the stream it was captured on)
            graph.replay()
            with torch.cuda.stream(other):
                block(eager)
            torch.cuda.synchronize()
            for n in ("y", "c", "s", "rw", "i", "r"):
                assert torch.equal(caught[n], eager[n]), n
    finally:
        cm.set_tile_policy(cm.TILE_AUTO)


@pytest.mark.parametrize("tile", [cm.TILE_DEC_GEMV, cm.TILE_ROWS32, cm.TILE_LDS_128, cm.TILE_128x256_OCC2, cm.TILE_W8])
@pytest.mark.parametrize("T, H", [(2, 256), (40, 416)])
def test_a_row_that_is_nan_stays_alone(T, H, tile):
    # a scale of 255 in one row's last block, a NaN code in another's first
    cm.set_tile_policy(tile)
    try:
        s = setup(T, H, 128, 4, 2, 0, BF, True, seed=3)
        s["x_scale"][0, H // 32 - 1] = 255
        s["x"][1, 0] = 0x7F
        out = run(s, 0, torch.empty(T, H, dtype=BF, device="cuda"))
        nan = torch.isnan(out)
        assert nan[:2].all() and not nan[2:].any()
    finally:
        cm.set_tile_policy(cm.TILE_AUTO)
