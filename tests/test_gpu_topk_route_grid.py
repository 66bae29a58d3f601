"""topk_route's choice on every width of a row, at scores that lie anywhere: the best
expert takes the last place of the keys' grid, whatever its roundings do."""
import numpy as np
import pytest
import torch

from test_gpu_topk_route import bias_of, call, logits_of

pytestmark = pytest.mark.gpu


def choice(l, k, bias, score):
    l = l.double().cpu().numpy()
    if score == "softmax":
        p = np.exp(l - l.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
    else:
        p = 1.0 / (1.0 + np.exp(-l))
    c = p if bias is None else p + bias.double().cpu().numpy()
    idx = np.argsort(-c, axis=1, kind="stable")[:, :k]
    return np.take_along_axis(p, idx, 1), idx


def check(l, k, bias, score, **kw):
    w, idx = choice(l, k, bias, score)
    got = call(l, k, bias, score=score, **kw)
    wrong = (got[1] != idx).any(1)
    assert not wrong.any(), f"{int(wrong.sum())} of {len(l)} rows, the first {int(wrong.argmax())}"
    w = w / w.sum(1, keepdims=True)
    assert (np.abs(got[0] - w) <= 2.0 ** -23 * w + 2.0 ** -149).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E", [8, 40, 60, 64, 96, 128, 256, 512])
@pytest.mark.parametrize("T", [300, 2040, 6000])
def test_the_best_expert_is_never_lost(T, E, score):
    k = min(E, 8)
    for seed, std in ((1, 1.0), (2, 0.1), (3, 4.0)):
        check(logits_of(T, E, seed=seed + E, std=std), k, None, score)
        check(logits_of(T, E, torch.bfloat16, seed=seed + E + 9, std=std), k, None, score)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("offset", [-100.0, -10.0, -1.0, -0.25, 0.25, 1.0, 10.0, 100.0, 1e4])
@pytest.mark.parametrize("T, E", [(300, 60), (300, 128), (6000, 64), (6000, 128), (6000, 256)])
def test_biases_far_from_zero(T, E, offset, score):
    # (f32 logits and biases: scores of one row differ by far more than the 64-bit
    # c's own rounding)
    check(logits_of(T, E, seed=E, std=1.0), 8, bias_of(E) + offset, score)
    check(logits_of(T, E, seed=E + 1, std=1.0), 8, torch.full((E,), offset, device="cuda"), score)
