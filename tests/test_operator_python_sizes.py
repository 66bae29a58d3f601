"""Sizes and options that the C entry points' 32-bit ints do not hold are refused in
Python, where ctypes would cut them to other values (no GPU needed: tensors without
memory)."""
import pytest
import torch

import candle_moe as cm

BIG = (1 << 32) + 1


def meta(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="meta")


def refused(who, call):
    with pytest.raises(cm.CandleMoeError, match=who + ": .* must fit 32 bits") as e:
        call()
    assert e.value.code == cm.CANDLE_MOE_ERR_INVALID


def route(T=4, E=8, k=2, **kw):
    i = meta(T, k, dtype=torch.int32)
    cm.topk_route(meta(T, E), meta(T, k), i, i, **kw)


@pytest.mark.parametrize("kw", [dict(T=BIG), dict(E=BIG), dict(num_groups=BIG), dict(topk_groups=BIG), dict(group_top=BIG),
                                dict(num_groups=-BIG)])
def test_route(kw):
    refused("topk_route", lambda: route(**kw))


@pytest.mark.parametrize("T, H", [(BIG, 1), (1, BIG)])
def test_norm(T, H):
    refused("add_rms_norm", lambda: cm.add_rms_norm(meta(T, H), meta(H), 1e-6, output=meta(T, H)))


def test_formats():
    u8 = torch.uint8
    refused("quantize_mxfp4", lambda: cm.quantize_mxfp4(meta(1, 32, BIG)))
    refused("quantize_mxfp4", lambda: cm.quantize_mxfp4(meta(BIG, 32, 1)))
    refused("dequantize_mxfp4", lambda: cm.dequantize_mxfp4(meta(1, BIG, 16, dtype=u8), meta(1, BIG, 1, dtype=u8), torch.float16))


@pytest.mark.parametrize("kw", [dict(T=BIG), dict(activation=BIG), dict(moe_type=BIG - 1)])
def test_moe(kw):
    T, H, I, E, k = kw.pop("T", 4), 32, 64, 2, 1
    nomic = kw.get("moe_type", 0) != 0
    q = lambda n, m: (meta(E, n, m // 2, dtype=torch.uint8), meta(E, n, m // 32, dtype=torch.uint8))  # noqa: E731
    gate, up, down = q(I, H), q(H, I) if nomic else q(I, H), (None, None) if nomic else q(H, I)
    x = meta(T, H, dtype=torch.bfloat16)
    refused("fused_moe_mxfp4", lambda: cm.fused_moe_mxfp4(
        x, gate[0], up[0], down[0], gate[1], up[1], down[1], meta(T, k), meta(T, k, dtype=torch.int32), x, E, k, **kw))
