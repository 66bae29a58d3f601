"""The operators around the expert products at sizes, layouts and values drawn over
their whole ranges, one seed a test, against their definitions in 64 bits."""
import random

import numpy as np
import pytest
import torch

import candle_moe as cm
import operator_reference as ref
from test_gpu_mxfp4 import BF, F16, run, setup
from test_gpu_mxfp4_sets import CODE, want
from test_gpu_rms_norm_extremes import check as check_norm
from test_gpu_topk_route import call

pytestmark = pytest.mark.gpu
INF = float("inf")


def log_int(rng, lo, hi):
    return int(round(2 ** rng.uniform(np.log2(lo), np.log2(hi))))


@pytest.mark.parametrize("seed", range(40))
def test_routes(seed):
    rng = random.Random(seed)
    E = rng.choice([rng.randint(1, 400), rng.choice([8, 32, 60, 64, 96, 128, 160, 256, 384, 512])])
    G = rng.choice([g for g in range(1, min(E, 64) + 1) if E % g == 0])
    tg, top = rng.randint(1, G), rng.randint(1, min(2, E // G))
    k = rng.randint(1, min(tg * (E // G), rng.choice([4, 8, 14, 20])))
    T = rng.choice([1, 7, 40, 300, 2100])
    kw = dict(score=rng.choice(["softmax", "sigmoid"]), num_groups=G, topk_groups=tg, group_top=top,
              renormalize=rng.random() < 0.6)
    dtype = rng.choice([torch.float32, torch.float32, BF, F16])
    g = torch.Generator().manual_seed(seed)
    l = torch.randn(T, E, generator=g) * rng.choice([0.1, 1, 4])
    for v in rng.sample([-INF, INF, float("nan"), torch.finfo(dtype).min, 0.0, -90.0, -700.0, 88.0], rng.randint(0, 3)):
        part = rng.choice([torch.rand(T, 1, generator=g) < 0.2, torch.rand(1, E, generator=g) < 0.2,
                           torch.rand(T, E, generator=g) < 0.1])
        l = torch.where(part, torch.tensor(v), l)
    b = None
    if rng.random() < 0.5:
        b = (torch.randn(E, generator=g) * rng.choice([0, 0.1, 1]) + rng.choice([0, 0, -1, 10])).cuda()
    l = l.to(dtype).cuda()
    got = call(l, k, b, **kw)
    w, i, ei = ref.route(l.double().cpu().numpy(), k, None if b is None else b.cpu().numpy(), **kw)
    assert np.array_equal(got[1], i) and np.array_equal(got[2], ei)
    assert np.array_equal(np.isnan(got[0]), np.isnan(w))
    off = np.abs(got[0].astype(np.float64) - w)[~np.isnan(w)]
    # (64-bit weights rounded once: test_gpu_topk_route_weights.py)
    assert (off <= ((2.0 ** -24 + 2.0 ** -40) * np.abs(w) + 2.0 ** -150)[~np.isnan(w)]).all()


@pytest.mark.parametrize("seed", range(30))
def test_norms(seed):
    rng = random.Random(seed)
    dtype = rng.choice([torch.float32, BF, F16])
    H = rng.choice([32 * log_int(rng, 1, 1024), log_int(rng, 1, 40000), 8 * log_int(rng, 1, 4096)])
    T = max(1, min(log_int(rng, 1, 3000), 10 ** 7 // H))
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, H, generator=g) * torch.exp2(2 * torch.randn(T, 1, generator=g))).to(dtype).cuda()
    r = torch.randn(T, H, generator=g).to(dtype).cuda() if rng.random() < 0.6 else None
    w = (1 + 0.2 * torch.randn(H, generator=g)).to(dtype).cuda()
    check_norm(x, w, rng.choice([0.0, 1e-6, 1e-5]), r, H % 32 == 0 and H <= 32768)


@pytest.mark.parametrize("seed", range(60))
def test_experts(seed):
    rng = random.Random(seed)
    E = rng.choice([1, 2, 4, 8, 8, 16, 60, 128, 300])
    k = rng.choice([1, 2, 3, 4, 8, 17])  # (a token may name an expert twice)
    H, I, T = 32 * log_int(rng, 1, 64), 32 * log_int(rng, 1, 48), log_int(rng, 1, 1500)
    while E * H * I > 1 << 26 or T * k * H * I > 1 << 35:
        E, T = max(1, E // 2), max(1, T // 2)
    moe_type, act, dtype, rows8 = rng.randint(0, 1), rng.randint(0, 2), rng.choice([BF, F16]), rng.random() < 0.4
    tile = rng.choice([cm.TILE_AUTO, cm.TILE_AUTO, cm.TILE_DEC_GEMV, cm.TILE_ROWS32, cm.TILE_LDS_128, cm.TILE_128x256_OCC2,
                       cm.TILE_W8])
    try:
        cm.set_tile_policy(tile)
        cm.set_combine_policy(rng.choice([cm.COMBINE_AUTO, cm.COMBINE_PAIRS, cm.COMBINE_EXPERT_SETS]))
        s = setup(T, H, I, E, min(k, E), moe_type, dtype, rows8, seed=seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        s["k"], s["idx"] = k, torch.randint(0, E, (T, k), generator=g, device="cuda").int()
        s["rw"] = torch.rand(T, k, generator=g, device="cuda") + 0.01
        gone = torch.rand(T, k, generator=g, device="cuda") < rng.choice([0.0, 0.1, 0.6])
        s["idx"][gone] = rng.choice([E, -7])
        sets = cm.fused_moe_mxfp4_path(T, H, I, E, k, CODE[dtype], moe_type, rows8) == "expert-set"
        y, far = want(s, act, sets, aligned=2.0 ** -12 if rows8 and dtype == BF else 0.0)
        # a dropped pair's weight is never looked at; a NaN row stays alone
        s["rw"][gone] = float("nan")
        nan = torch.rand(T, generator=g, device="cuda") < 0.1
        s["x"][nan, 0] = 127 if rows8 else float("nan")
        out = torch.full((T + 1, H), 5.0, dtype=dtype, device="cuda")
        out[:T] = torch.randn(T, H, generator=g, device="cuda").to(dtype)
        accumulate = rng.random() < 0.3
        if accumulate:
            y = y + out[:T].double()
            far = far + ref.HALF[dtype] * (y.abs() + far)
        run(s, act, out[:T], accumulate=accumulate)
        ref.within(out[:T][~nan], y[~nan], far[~nan])
        assert (out[T] == 5).all()
    finally:
        cm.set_tile_policy(cm.TILE_AUTO)
        cm.set_combine_policy(cm.COMBINE_AUTO)
