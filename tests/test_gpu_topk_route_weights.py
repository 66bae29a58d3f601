"""topk_route's weights: 64-bit values rounded to f32 once, in every form of a row.
Their own 64-bit roundings, of the exponentials (2^-52 each), of a sum of up to 1024
of them and of the divisions, stay below 2^-40 of a weight; the rounding is at most
2^-24 of it (2^-150 below the normal range)."""
import numpy as np
import pytest
import torch

import operator_reference as ref
from test_gpu_topk_route import bias_of, call, logits_of

pytestmark = pytest.mark.gpu


def check_once_rounded(l, k, bias=None, **kw):
    got = call(l, k, bias, **kw)
    w, i, _ = ref.route(l.double().cpu().numpy(), k, None if bias is None else bias.cpu().numpy(), **kw)
    assert np.array_equal(got[1], i)
    off = np.abs(got[0].astype(np.float64) - w)
    assert (off <= (2.0 ** -24 + 2.0 ** -40) * np.abs(w) + 2.0 ** -150).all(), float((off / np.abs(w)).max() * 2.0 ** 24)
    return got


@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T, E, k", [(1, 8, 3), (5, 64, 8), (40, 128, 8), (33, 256, 8), (17, 512, 8), (9, 1000, 8), (9, 1024, 8),
                                     (2100, 64, 8), (2100, 128, 8), (2100, 256, 8), (2100, 512, 8), (3, 512, 70)])
def test_rounded_once(T, E, k, score, renorm):
    for seed, dtype in ((T, torch.float32), (E, torch.bfloat16)):
        check_once_rounded(logits_of(T, E, dtype, seed=seed), k, score=score, renormalize=renorm, scale=2.5)
    check_once_rounded(logits_of(T, E, seed=7), k, bias_of(E), score=score, renormalize=renorm)


@pytest.mark.parametrize("offset", [3.0, 4.2, 5.1, 5.6, 6.3, 7.0, 30.0, 87.5, 100.0])
@pytest.mark.parametrize("T, E", [(4, 256), (4, 1024), (2100, 256), (2100, 512)])
def test_many_equal_tail_logits(T, E, offset):
    # one expert ahead, the others near alike: every f32 rounding of the tail's
    # exponentials would go the same way
    l = logits_of(T, E, seed=3, std=1e-4) - offset + 0.5
    l[:, ::97] += 0.01 * torch.arange(1, l[:, ::97].shape[1] + 1, device="cuda")
    l[torch.arange(T), torch.arange(T) % E] = 0.5 + torch.arange(T, device="cuda") / 4096
    check_once_rounded(l, 8, score="softmax", renormalize=False)


def test_a_row_has_the_same_weights_in_every_batch():
    # 64 lanes of a row in a small batch, 16 in a large one; sums of other orders
    # differ by 2^-45 at most, so no f32 weight of these rows does
    l = logits_of(2100, 256, seed=5)
    for score in ("softmax", "sigmoid"):
        kw = dict(score=score, renormalize=False)
        many = call(l, 8, None, **kw)
        few = call(l[:100].contiguous(), 8, None, **kw)
        assert np.array_equal(many[0][:100], few[0]) and np.array_equal(many[1][:100], few[1])
