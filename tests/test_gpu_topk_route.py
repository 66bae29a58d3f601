"""topk_route against its definition in 64 bits: the choice exactly, the weights
to a rounding of f32 (2^-24) and of the 64-bit scores' own."""
import numpy as np
import pytest
import torch

import candle_moe as cm
import operator_reference as ref

pytestmark = pytest.mark.gpu


def call(logits, k, bias=None, **kw):
    T = logits.shape[0]
    w = torch.full((T, k), float("nan"), device="cuda")
    i, ei = (torch.full((T, k), -1, dtype=torch.int32, device="cuda") for _ in range(2))
    cm.topk_route(logits, w, i, ei, bias=bias, **kw)
    torch.cuda.synchronize()
    return w.cpu().numpy(), i.cpu().numpy(), ei.cpu().numpy()


def check(logits, k, bias=None, **kw):
    got = call(logits, k, bias, **kw)
    w, i, ei = ref.route(logits.double().cpu().numpy(), k, None if bias is None else bias.cpu().numpy(), **kw)
    assert np.array_equal(got[1], i)
    assert np.array_equal(got[2], ei)
    assert np.array_equal(np.isnan(got[0]), np.isnan(w))
    off = np.abs(got[0] - w)
    # the weights of a softmax that is not renormalised hold a sum of f32 exponentials:
    # one ulp (2^-23) each and three f32 additions, 2^-22 with them; the others 64-bit
    # values rounded once
    u = 2.0 ** -23 if kw.get("renormalize", True) or kw.get("score") == "sigmoid" else 2.0 ** -21
    assert (off[~np.isnan(w)] <= (u * np.abs(w) + 2.0 ** -149)[~np.isnan(w)]).all()


def logits_of(T, E, dtype=torch.float32, seed=1, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, E, generator=g) * std).to(dtype).cuda()


def bias_of(E, seed=2, std=0.1):
    return (torch.randn(E, generator=torch.Generator().manual_seed(seed)) * std).cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T, E, k", [(1, 1, 1), (1, 8, 8), (3, 60, 4), (5, 64, 6), (130, 65, 8), (7, 128, 8), (66, 160, 6),
                                     (33, 256, 8), (9, 384, 20), (3, 512, 70), (5, 1000, 8), (2, 1024, 1024)])
def test_choice_and_weights(T, E, k, score, dtype):
    l = logits_of(T, E, dtype, seed=T + E)
    check(l, k, score=score)
    check(l, k, bias_of(E), score=score, renormalize=False, scale=2.5)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E, G, tg, top, k", [(256, 8, 4, 2, 8), (256, 8, 4, 1, 8), (160, 8, 3, 1, 6), (64, 1, 1, 2, 4),
                                              (64, 64, 8, 1, 8), (60, 4, 2, 2, 30), (96, 3, 1, 2, 32), (512, 16, 16, 2, 8),
                                              (1024, 32, 4, 2, 8), (1000, 40, 7, 2, 9), (8, 4, 2, 2, 4), (12, 4, 3, 2, 9)])
def test_groups(E, G, tg, top, k, score):
    kw = dict(score=score, num_groups=G, topk_groups=tg, group_top=top)
    check(logits_of(67, E, seed=E + G), k, bias_of(E), **kw)
    check(logits_of(5, E, torch.bfloat16, seed=E), k, **kw)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E, G, tg", [(64, 1, 1), (128, 8, 3), (256, 8, 4), (512, 8, 2)])
def test_ties_go_to_the_lower_index(E, G, tg, score):
    l = torch.randint(-2, 3, (40, E), generator=torch.Generator().manual_seed(E)).float().cuda()
    l[0] = 0.0
    kw = dict(score=score, num_groups=G, topk_groups=tg, group_top=2 if G > 1 else 1)
    check(l, 8, **kw)
    check(l, 8, torch.zeros(E, device="cuda"), **kw)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E, G, tg", [(64, 1, 1), (256, 8, 4)])
def test_scores_that_differ_in_the_last_bits(E, G, tg, score):
    # neighbouring f32 logits, and biases that nearly undo the difference of scores
    base = logits_of(50, E, seed=3)
    near = torch.nextafter(base[:, : E // 2], torch.full((), 9.0, device="cuda"))
    l = torch.cat((base[:, : E // 2], near), 1)
    kw = dict(score=score, num_groups=G, topk_groups=tg, group_top=1)
    check(l, 8, **kw)
    p = torch.sigmoid(l[0].double()) if score == "sigmoid" else torch.softmax(l[0].double(), 0)
    check(l, 8, (0.25 - p).float(), **kw)  # row 0: all c within an f32 rounding of 0.25


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E, G, tg", [(60, 1, 1), (64, 1, 1), (128, 1, 1), (256, 8, 4)])
def test_masks_and_what_is_not_finite(E, G, tg, score):
    inf, nan = float("inf"), float("nan")
    l = logits_of(14, E, seed=4)
    l[0] = -inf
    l[1, 3:] = -inf
    l[2] = torch.finfo(torch.float32).min
    l[3, ::2] = torch.finfo(torch.float32).min
    l[4, 5] = nan
    l[5] = nan
    l[6, 7] = inf
    l[7] = inf
    l[8, :] = -inf
    l[8, E - 1] = 0.0
    l[9, 0], l[9, 1] = inf, -inf
    l[10] *= 1e30
    l[11] *= 1e-30
    l[12] = -90.0
    l[12, 4:9] = torch.tensor([-90.0, -89.0, -88.0, -87.0, -86.0])
    kw = dict(score=score, num_groups=G, topk_groups=tg, group_top=1)
    for renorm in (True, False):
        check(l, 4, renormalize=renorm, **kw)
    b = bias_of(E)
    b[1], b[2], b[3] = -inf, nan, -1e30
    check(l, 4, b, **kw)
    check(l, 4, torch.full((E,), -inf, device="cuda"), **kw)


def test_large_batch_and_past_the_last_row():
    T, E, k = 4099, 256, 8
    w = torch.full((T + 3, k), 7.0, device="cuda")
    i, ei = (torch.full((T + 3, k), 7, dtype=torch.int32, device="cuda") for _ in range(2))
    l = logits_of(T, E, seed=6)
    kw = dict(score="sigmoid", num_groups=8, topk_groups=4, group_top=2, scale=2.5)
    cm.topk_route(l, w[:T], i[:T], ei[:T], bias=bias_of(E), **kw)
    want = ref.route(l.cpu().double().numpy(), k, bias_of(E).cpu().numpy(), **kw)
    assert np.array_equal(i[:T].cpu().numpy(), want[1]) and np.array_equal(ei[:T].cpu().numpy(), want[2])
    for t in (w, i, ei):
        assert (t[T:] == 7).all()


def test_unaligned_logits():
    l = logits_of(9, 128, torch.bfloat16, seed=7)
    flat = torch.zeros(9 * 128 + 1, dtype=torch.bfloat16, device="cuda")
    flat[1:] = l.flatten()
    check(flat[1:].view(9, 128), 8)
    flat = torch.zeros(9 * 256 + 3, device="cuda")
    flat[3:] = logits_of(9, 256, seed=8).flatten()
    check(flat[3:].view(9, 256), 8, bias_of(256), num_groups=8, topk_groups=4, group_top=2, score="sigmoid")


def test_graph_on_another_stream():
    T, E, k = 37, 256, 8
    l = logits_of(T, E, seed=9)
    w = torch.zeros((T, k), device="cuda")
    i, ei = (torch.zeros((T, k), dtype=torch.int32, device="cuda") for _ in range(2))
    kw = dict(bias=bias_of(E), score="sigmoid", num_groups=8, topk_groups=4, group_top=2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        cm.topk_route(l, w, i, ei, **kw)
    for seed in (10, 11, 12):
        l.copy_(logits_of(T, E, seed=seed))
        g.replay()
        torch.cuda.synchronize()
        again = call(l, k, kw["bias"], **{n: v for n, v in kw.items() if n != "bias"})
        assert np.array_equal(again[0], w.cpu().numpy()) and np.array_equal(again[1], i.cpu().numpy())
        check(l, k, **kw)
