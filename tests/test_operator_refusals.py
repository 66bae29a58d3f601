"""What topk_route, add_rms_norm and the MXFP4 calls refuse, before anything is
launched (no GPU needed): sizes at the C entry points, tensors in Python."""
import ctypes

import pytest
import torch

import candle_moe as cm

P = ctypes.c_void_p(4096)  # never read
INVALID, UNSUPPORTED = cm.CANDLE_MOE_ERR_INVALID, cm.CANDLE_MOE_ERR_UNSUPPORTED


def route(T=4, E=16, k=2, dtype=2, score=0, G=1, tg=1, top=1, w=P):
    return cm.lib().candle_moe_topk_route(P, dtype, None, w, P, P, E, T, k, score, G, tg, top, 1, 1.0, None)


@pytest.mark.parametrize("bad", [dict(T=-1), dict(E=0), dict(E=1025), dict(k=0), dict(k=17), dict(dtype=3), dict(score=2),
                                 dict(score=-1), dict(G=0), dict(G=3), dict(G=65, E=65), dict(G=4, tg=5), dict(G=4, tg=0),
                                 dict(top=0), dict(top=3), dict(G=16, tg=2, top=2), dict(G=4, tg=1, k=5), dict(w=None)])
def test_route_refuses(bad):
    assert route(**bad) == INVALID
    assert "topk_route" in cm.last_error()


def test_nothing_to_do_is_fine():
    assert route(T=0, w=None) == 0
    assert norm(T=0, x=None) == 0
    assert moe(T=0, x=None) == 0
    assert cm.lib().candle_moe_quantize_mxfp4(None, 2, 0, 32, 8, 1, None, None, None) == 0
    assert cm.lib().candle_moe_dequantize_mxfp4(None, None, 2, 0, 32, None, 1, None) == 0


def norm(T=4, H=64, eps=1e-6, dtype=1, x=P, w=P, out=P, codes=None, scales=None):
    return cm.lib().candle_moe_add_rms_norm(x, None, w, None, out, codes, scales, T, H, eps, dtype, None)


@pytest.mark.parametrize("bad, code", [
    (dict(T=-1), INVALID), (dict(H=0), INVALID), (dict(dtype=3), INVALID), (dict(eps=-1.0), INVALID),
    (dict(eps=float("nan")), INVALID), (dict(x=None), INVALID), (dict(w=None), INVALID), (dict(out=None), INVALID),
    (dict(codes=P), INVALID), (dict(scales=P), INVALID), (dict(H=48, codes=P, scales=P), UNSUPPORTED),
    (dict(H=32800, codes=P, scales=P), UNSUPPORTED),
    (dict(x=ctypes.c_void_p(4098), codes=P, scales=P), UNSUPPORTED)])
def test_norm_refuses(bad, code):
    assert norm(**bad) == code
    assert "add_rms_norm" in cm.last_error()


def moe(T=4, H=64, I=96, E=8, k=2, act=0, mt=0, dtype=1, x=P, gate=P, down=P, down_s=P, out=P):
    return cm.lib().candle_moe_fused_moe_mxfp4(x, None, gate, P, down, P, P, down_s, P, P, out, T, H, I, E, k, act, mt,
                                               dtype, 0, None)


@pytest.mark.parametrize("bad, code", [
    (dict(T=-1), INVALID), (dict(E=0), INVALID), (dict(E=4097), INVALID), (dict(k=0), INVALID), (dict(act=3), INVALID),
    (dict(mt=2), INVALID), (dict(dtype=2), UNSUPPORTED), (dict(H=48), UNSUPPORTED), (dict(I=80), UNSUPPORTED),
    (dict(H=0), UNSUPPORTED), (dict(T=1 << 30, k=2), INVALID), (dict(x=None), INVALID), (dict(gate=None), INVALID),
    (dict(down=None), INVALID), (dict(down_s=None), INVALID), (dict(out=None), INVALID),
    (dict(x=ctypes.c_void_p(4104)), UNSUPPORTED), (dict(out=ctypes.c_void_p(4104)), UNSUPPORTED),
    (dict(T=1 << 24, H=64), UNSUPPORTED)])
def test_moe_refuses(bad, code):
    assert moe(**bad) == code
    assert "fused_moe_mxfp4" in cm.last_error()


def test_formats_refuse():
    L = cm.lib()
    for args, code in (((P, 3, 2, 32, 8, 1, P, P, None), INVALID), ((P, 2, -1, 32, 8, 1, P, P, None), INVALID),
                       ((P, 2, 2, 48, 8, 1, P, P, None), UNSUPPORTED), ((None, 2, 2, 32, 8, 1, P, P, None), INVALID),
                       ((P, 2, 2, 32, 8, 1, ctypes.c_void_p(4100), P, None), UNSUPPORTED)):
        assert L.candle_moe_quantize_mxfp4(*args) == code and "quantize_mxfp4" in cm.last_error()
    for args, code in (((P, P, 2, 8, 32, P, 3, None), INVALID), ((P, P, 2, 8, 40, P, 1, None), UNSUPPORTED),
                       ((P, None, 2, 8, 32, P, 1, None), INVALID), ((P, P, 2, -8, 32, P, 1, None), INVALID),
                       ((P, P, 2, 8, 32, ctypes.c_void_p(4100), 1, None), UNSUPPORTED)):
        assert L.candle_moe_dequantize_mxfp4(*args) == code and "dequantize_mxfp4" in cm.last_error()


# ----------------------------------------------------------- tensors in Python
def route_tensors(T=3, E=8, k=2):
    return [torch.zeros(T, E), torch.zeros(T, k), torch.zeros(T, k, dtype=torch.int32),
            torch.zeros(T, k, dtype=torch.int32)]


@pytest.mark.parametrize("change, word", [
    (lambda t: t, "on the GPU"), (lambda t: [t[0].double()] + t[1:], "logits must be"),
    (lambda t: [torch.zeros(8, 3).t()] + t[1:], "contiguous"), (lambda t: [t[0][0]] + t[1:], r"\[T, E\]"),
    (lambda t: [t[0], t[1].half(), t[2], t[3]], "topk_weight must be"), (lambda t: [t[0], t[1], t[2].long(), t[3]], "topk_indices"),
    (lambda t: [t[0], t[1], t[2], t[3][:, :1]], "token_expert_indices")])
def test_route_tensors(change, word):
    with pytest.raises(cm.CandleMoeError, match=word):
        cm.topk_route(*change(route_tensors()))


def test_route_words():
    with pytest.raises(cm.CandleMoeError, match="softmax or sigmoid"):
        cm.topk_route(*route_tensors(), score="relu")
    with pytest.raises(cm.CandleMoeError, match="bias"):
        cm.topk_route(*route_tensors(), bias=torch.zeros(7))


@pytest.mark.parametrize("kw, word", [
    (dict(), "on the GPU"), (dict(weight=torch.ones(32)), "weight"), (dict(output=torch.zeros(3, 64).half()), "output"),
    (dict(residual=torch.zeros(2, 64)), "residual"), (dict(codes=torch.zeros(3, 64, dtype=torch.uint8)), "scales is missing"),
    (dict(scales=torch.zeros(3, 2, dtype=torch.uint8)), "codes is missing"),
    (dict(codes=torch.zeros(3, 64, dtype=torch.uint8), scales=torch.zeros(3, 3, dtype=torch.uint8)), "scales must be"),
    (dict(residual_output=torch.zeros(64, 3).t()), "contiguous")])
def test_norm_tensors(kw, word):
    kw = {"output": torch.zeros(3, 64), "weight": torch.ones(64), **kw}
    with pytest.raises(cm.CandleMoeError, match=word):
        cm.add_rms_norm(torch.zeros(3, 64), kw.pop("weight"), 1e-6, **kw)


def moe_tensors(T=3, H=64, I=32, E=4, k=2):
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)  # noqa: E731
    return dict(input=torch.zeros(T, H).bfloat16(), gate_q=u8(E, I, H // 2), up_q=u8(E, I, H // 2), down_q=u8(E, H, I // 2),
                gate_scale=u8(E, I, H // 32), up_scale=u8(E, I, H // 32), down_scale=u8(E, H, I // 32),
                routing_weights=torch.zeros(T, k), expert_indices=torch.zeros(T, k, dtype=torch.int32),
                output=torch.zeros(T, H).bfloat16(), num_experts=E, top_k=k)


@pytest.mark.parametrize("kw, word", [
    (dict(), "on the GPU"), (dict(down_q=None), "down_q is missing"), (dict(moe_type=1), "no down_q"),
    (dict(output=torch.zeros(3, 64)), "output"), (dict(input=torch.zeros(3, 64).half()), "input"),
    (dict(input_scale=torch.zeros(3, 2, dtype=torch.uint8)), "input must be"),
    (dict(input=torch.zeros(3, 48).bfloat16()), "multiples of 32"), (dict(num_experts=5), "gate_q"),
    (dict(routing_weights=torch.zeros(3, 2).half()), "routing_weights"), (dict(top_k=3), "routing_weights"),
    (dict(gate_scale=torch.zeros(4, 32, 2)), "gate_scale")])
def test_moe_tensors(kw, word):
    with pytest.raises(cm.CandleMoeError, match=word):
        cm.fused_moe_mxfp4(**{**moe_tensors(), **kw})


def test_format_tensors():
    with pytest.raises(cm.CandleMoeError, match="contiguous"):
        cm.quantize_mxfp4(torch.zeros(4, 32))
    with pytest.raises(cm.CandleMoeError, match="on the GPU"):
        cm.quantize_mxfp4(torch.zeros(2, 32, 8))
    with pytest.raises(cm.CandleMoeError, match="scales"):
        cm.dequantize_mxfp4(torch.zeros(2, 8, 32, dtype=torch.uint8), torch.zeros(2, 8, 1, dtype=torch.uint8), torch.float32)
