"""MXFP4 weights and the MoE over them. The formats bit for bit; the MoE against
64 bits within what operator_reference.moe derives from its roundings."""
import pytest
import torch

import candle_moe as cm
import operator_reference as ref

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16


def randn(*shape, seed, std=1.0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std


# -------------------------------------------------------------------- formats
def test_dequantize_every_code_and_scale():
    codes = torch.arange(16, dtype=torch.uint8).repeat(2)
    packed = (codes[0::2] | (codes[1::2] << 4)).view(1, 1, 16).expand(1, 256, 16).contiguous().cuda()
    scales = torch.arange(256, dtype=torch.int32).to(torch.uint8).view(1, 256, 1).cuda()
    want = ref.from_mxfp4(packed, scales)
    for dt in (torch.float32, BF, F16):
        got = cm.dequantize_mxfp4(packed, scales, dt)
        exact = want.to(torch.float32).to(dt)  # (exact in f32)
        assert torch.equal(torch.isnan(got), torch.isnan(exact))
        assert torch.equal(got[~torch.isnan(got)], exact[~torch.isnan(exact)])


@pytest.mark.parametrize("dtype", [torch.float32, F16, BF])
@pytest.mark.parametrize("E, K, N", [(1, 32, 1), (3, 96, 40), (2, 256, 33), (2, 64, 129)])
def test_quantize(E, K, N, dtype):
    w = randn(E, K, N, seed=K + N, std=0.05)
    w[0, :32, 0] = 0.0
    w[0, :, N - 1] = 2.0 ** -10
    # ties and borders of a block whose largest is 6 * 2^0
    w[E - 1, :16, N // 2] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5,
                                          -5.0, 0.2])
    w = w.to(dtype).cuda()
    codes, scales = cm.quantize_mxfp4(w)
    wc, ws = ref.mxfp4(w.transpose(1, 2).contiguous())
    assert torch.equal(scales, ws) and torch.equal(codes, wc)
    c2, s2 = cm.quantize_mxfp4(w.transpose(1, 2).contiguous(), input_kn=False)
    assert torch.equal(s2, ws) and torch.equal(c2, wc)


def test_quantize_extremes():
    w = torch.zeros(1, 7, 32)
    w[0, 0, 3] = 3.4e38
    w[0, 1, 3] = 1e-45
    w[0, 2, 0], w[0, 2, 1] = 6.0, 6.0 * (1 - 2.0 ** -23)
    w[0, 3, 0] = 6.0 * (1 + 2.0 ** -22)
    w[0, 4, 9] = float("nan")
    w[0, 5, 9] = float("-inf")
    w[0, 6] = -1e-40
    w = w.cuda()
    codes, scales = cm.quantize_mxfp4(w, input_kn=False)
    wc, ws = ref.mxfp4(w)
    assert torch.equal(scales, ws) and torch.equal(codes, wc)
    assert scales[0, :, 0].tolist()[2:6] == [127, 128, 255, 255]


# ------------------------------------------------------------------------ MoE
def setup(T, H, I, E, k, moe_type, dtype, rows8, seed=1, dropped=0.0, skew=False):
    dev = "cuda"
    gate = ref.mxfp4(randn(E, I, H, seed=seed, std=0.05).to(dev))
    up = ref.mxfp4(randn(*((E, I, H) if moe_type == 0 else (E, H, I)), seed=seed + 1, std=0.05).to(dev))
    down = ref.mxfp4(randn(E, H, I, seed=seed + 2, std=0.05).to(dev)) if moe_type == 0 else (None, None)
    l = randn(T, E, seed=seed + 3)
    if skew:
        l[:, 0] += 6
    p, idx = torch.softmax(l, -1).topk(k, -1)
    rw = (p / p.sum(-1, keepdim=True)).cuda()
    if dropped:
        idx = torch.where(torch.rand(T, k, generator=torch.Generator().manual_seed(seed + 4)) < dropped, E, idx)
    idx = idx.to(torch.int32).cuda()
    x = randn(T, H, seed=seed + 5).to(dev)
    scale = None
    if rows8:
        b = x.double().unflatten(-1, (-1, 32))
        scale = ref.mx_scale(b.abs().amax(-1), 448.0)
        x = (b / ref.scale_value(scale).unsqueeze(-1)).flatten(-2).float().to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        x = x.to(dtype)
    return dict(x=x, x_scale=scale, gate=gate, up=up, down=down, rw=rw, idx=idx, E=E, k=k, moe_type=moe_type, dtype=dtype)


def run(s, act, out, accumulate=False):
    cm.fused_moe_mxfp4(s["x"], s["gate"][0], s["up"][0], s["down"][0], s["gate"][1], s["up"][1], s["down"][1], s["rw"],
                       s["idx"], out, s["E"], s["k"], activation=act, moe_type=s["moe_type"], input_scale=s["x_scale"],
                       accumulate=accumulate)
    return out


def want(s, act, aligned=0.0):
    x = s["x"] if s["x_scale"] is None else ref.from_mxfp8(s["x"], s["x_scale"])
    w = [ref.from_mxfp4(*q) if q[0] is not None else None for q in (s["gate"], s["up"], s["down"])]
    return ref.moe(x, *w, s["rw"], s["idx"], act, s["moe_type"], s["dtype"], aligned=aligned)


def check(s, act, what="", aligned=0.0):
    T, H = s["x"].shape
    out = torch.full((T, H), float("nan"), dtype=s["dtype"], device="cuda")
    ref.within(run(s, act, out), *want(s, act, aligned), what)
    return out


SIZES = [(1, 32, 32, 1, 1), (1, 256, 128, 8, 2), (2, 96, 160, 4, 3), (5, 2048, 768, 16, 4), (16, 512, 256, 8, 2),
         (17, 128, 96, 3, 3), (33, 416, 288, 8, 2), (64, 256, 512, 4, 1), (130, 288, 96, 5, 2), (300, 512, 256, 4, 2),
         (700, 256, 384, 8, 2)]


@pytest.mark.parametrize("rows8", [False, True])
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("moe_type", [0, 1])
@pytest.mark.parametrize("T, H, I, E, k", SIZES)
def test_moe(T, H, I, E, k, moe_type, dtype, rows8):
    s = setup(T, H, I, E, k, moe_type, dtype, rows8, seed=T + H)
    check(s, (T + moe_type) % 3)


@pytest.mark.parametrize("rows8", [False, True])
@pytest.mark.parametrize("T", [1, 9, 40, 257])
def test_dropped_pairs_skew_and_empty(T, rows8):
    check(setup(T, 256, 128, 8, 4, 0, BF, rows8, dropped=0.3), 0)
    check(setup(T, 256, 128, 8, 2, 0, BF, rows8, skew=True), 0)
    s = setup(T, 256, 128, 8, 2, 1, BF, rows8)
    s["idx"].fill_(8)
    assert (check(s, 1) == 0).all()
    s["idx"].fill_(-1)  # (as u32: past every expert)
    assert (check(s, 1) == 0).all()
    s["idx"].fill_(3)  # one expert, in every slot
    check(s, 1)


@pytest.mark.parametrize("rows8", [False, True])
@pytest.mark.parametrize("T", [1, 12, 200])
def test_accumulate_and_rows_past_the_batch(T, rows8):
    s = setup(T, 256, 160, 8, 2, 0, BF, rows8)
    big = randn(T + 2, 256, seed=9).to(BF).cuda()
    before = big.clone()
    y, far = want(s, 0)
    run(s, 0, big[:T], accumulate=True)
    total = before[:T].double() + y
    ref.within(big[:T], total, far + 2.0 ** -8 * (total.abs() + far))
    assert torch.equal(big[T:], before[T:])


@pytest.mark.parametrize("T", [3, 50, 300])
def test_a_weight_that_is_nan_stays_in_its_expert(T):
    s = setup(T, 256, 128, 4, 1, 0, BF, False)
    s["gate"][1][2, 7, 1] = 255
    out = run(s, 0, torch.zeros(T, 256, dtype=BF, device="cuda"))
    hit = (s["idx"] == 2).any(1)
    assert torch.isnan(out[hit]).all() and not torch.isnan(out[~hit]).any()


@pytest.mark.parametrize("dtype", [BF, F16])
def test_scales_far_apart(dtype):
    # blocks from 2^-20 to 2^6 in one column: each product keeps its own size
    s = setup(11, 256, 128, 4, 2, 0, dtype, False)
    for q in (s["gate"], s["up"], s["down"]):
        q[1].copy_((107 + (torch.arange(q[1].numel(), device="cuda") * 7) % 15).to(torch.uint8).view_as(q[1]))
    s["gate"][1][0, 0, 0] = 0
    check(s, 2)


def test_same_bits_again_and_on_another_stream():
    for T in (3, 40, 300):
        s = setup(T, 256, 256, 8, 2, 0, BF, False)
        outs = [torch.empty(T, 256, dtype=BF, device="cuda") for _ in range(3)]
        run(s, 0, outs[0])
        torch.cuda.synchronize()
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            run(s, 0, outs[1])
        run(s, 0, outs[2])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("rows8", [False, True])
def test_graphs_of_smaller_batches_after_one_large_call(rows8):
    H, I, E, k = 256, 384, 8, 2
    st = torch.cuda.Stream()
    sets = {T: setup(T, H, I, E, k, 0, BF, rows8, seed=T) for T in (700, 300, 40, 8, 1)}
    outs = {T: torch.empty(T, H, dtype=BF, device="cuda") for T in sets}
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        run(sets[700], 0, outs[700])
    torch.cuda.synchronize()
    graphs = {}
    for T in (300, 40, 8, 1):
        graphs[T] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graphs[T], stream=st):
            run(sets[T], 0, outs[T])
    for _ in range(3):
        for T, g in graphs.items():
            sets[T]["x"].copy_(sets[T]["x"].flip(0))
            eager = run(sets[T], 0, torch.empty_like(outs[T]))
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(eager, outs[T]), T
    ref.within(outs[8], *want(sets[8], 0))


def test_refused_capture_launches_nothing():
    cm.trim_workspaces()
    s = setup(4, 256, 128, 8, 2, 0, BF, False)
    out = torch.zeros(4, 256, dtype=BF, device="cuda")
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        with pytest.raises(cm.CandleMoeError) as e:
            run(s, 0, out)
        out.add_(1)
    assert e.value.code == cm.CANDLE_MOE_ERR_WORKSPACE
    g.replay()
    torch.cuda.synchronize()
    assert (out == 1).all()


# ---------------------------------------------------------- all of them in turn
@pytest.mark.parametrize("rows8", [False, True])
@pytest.mark.parametrize("T", [1, 5, 150])
def test_a_block_from_its_residual_to_its_experts(T, rows8):
    """add_rms_norm, the router's logits, topk_route, fused_moe_mxfp4 over
    quantize_mxfp4's weights: each against its own definition on the one before's
    outputs."""
    H, I, E, k = 512, 256, 32, 4
    x, r = (randn(T, H, seed=i, std=i).to(BF).cuda() for i in (1, 2))
    w = (1 + 0.1 * randn(H, seed=3)).to(BF).cuda()
    y, ro = torch.empty_like(x), torch.empty_like(x)
    codes, scales = (torch.empty(T, n, dtype=torch.uint8, device="cuda") for n in (H, H // 32))
    cm.add_rms_norm(x, w, 1e-6, residual=r, residual_output=ro, output=y, codes=codes, scales=scales)
    logits = y.float() @ randn(E, H, seed=4, std=0.05).cuda().t()
    rw = torch.empty(T, k, device="cuda")
    idx, ei = (torch.empty(T, k, dtype=torch.int32, device="cuda") for _ in range(2))
    kw = dict(score="sigmoid", num_groups=4, topk_groups=2, group_top=2, scale=2.5)
    bias = randn(E, seed=5, std=0.1).cuda()
    cm.topk_route(logits, rw, idx, ei, bias=bias, **kw)
    mats = [randn(E, a, b, seed=s, std=0.05).to(BF).cuda() for a, b, s in ((H, I, 6), (H, I, 7), (I, H, 8))]
    (g, gs), (u, us), (d, ds) = (cm.quantize_mxfp4(m) for m in mats)
    out = ro.clone()  # the layer adds into the residual stream
    cm.fused_moe_mxfp4(codes if rows8 else y, g, u, d, gs, us, ds, rw, idx, out, E, k,
                       input_scale=scales if rows8 else None)
    ww, wi, _ = ref.route(logits.double().cpu().numpy(), k, bias.cpu().numpy(), **kw)
    assert (idx.cpu().numpy() == wi).all()
    rows = ref.from_mxfp8(codes, scales) if rows8 else y
    mo, far = ref.moe(rows, ref.from_mxfp4(g, gs), ref.from_mxfp4(u, us), ref.from_mxfp4(d, ds), rw, idx, 0, 0, BF)
    total = ro.double() + mo
    ref.within(out, total, far + 2.0 ** -8 * (total.abs() + far))
    _, yw = ref.norm(x, w, 1e-6, r)
    ref.within(y, yw, 2.0 ** -8 * yw.abs() * 1.001 + 2.0 ** -17 * yw.abs())
