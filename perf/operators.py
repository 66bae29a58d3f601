"""The operators around and inside a mixture-of-experts layer, measured.

  route  topk_route: scores of the experts (softmax or sigmoid), a bias that
         balances their load, a choice of groups, the top k and their weights
  norm   add_rms_norm: the residual's addition, the root-mean-square norm and
         its 8-bit form (e4m3 values, one power of two per 32: MXFP8)
  moe    fused_moe_mxfp4: the experts' products over 4-bit weights (e2m1
         values, one power of two per 32: MXFP4), on 16-bit or 8-bit rows

`own` says which form `run` takes: the framework's calls, or the formulas in
elementary torch operations. Model sizes are the repository's own: Qwen3
(H 4096, I 1536, 8 experts, top 2), Qwen3-30B-A3B (H 2048, I 768, 128 experts,
top 8); others are generic.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
ACTS = {"silu": 0, "gelu": 1, "relu": 2}
EPS = 1e-6
LOWEST = -1.7976931348623157e308  # the least finite f64

QWEN3 = dict(H=4096, I=1536, E=8, k=2, act="silu", moe_type=0)
Q30B = dict(H=2048, I=768, E=128, k=8, act="silu", moe_type=0)
EMBED = dict(H=768, I=2048, E=8, k=2, act="gelu", moe_type=1)


def _package():
    path = os.path.join(os.getcwd(), "candle-moe_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import candle_moe

    return candle_moe


def _route(T, E, k, score, bias, groups, topk_groups, group_top, renorm, scale, dtype):
    return dict(kind="route", T=T, E=E, k=k, score=score, bias=bias, groups=groups, topk_groups=topk_groups,
                group_top=group_top, renorm=renorm, scale=scale, dtype=dtype)


def _norm(T, H, dtype, residual, wide, mx):
    return dict(kind="norm", T=T, H=H, dtype=dtype, residual=residual, wide=wide, mx=mx)


def _moe(model, T, dtype, rows="16", skew=False, dropped=False):
    return dict(kind="moe", T=T, dtype=dtype, rows=rows, skew=skew, dropped=dropped, **model)


def listed():
    return [
        # one token of a decode step: latency only
        dict(name="route_decode_1", **_route(1, 128, 8, "softmax", False, 1, 1, 1, True, 1.0, "bf16")),
        # a ragged prefill chunk of a model whose router balances by a bias
        dict(name="route_groups_4099", **_route(4099, 256, 8, "sigmoid", True, 8, 4, 2, True, 2.5, "f32")),
        # the largest prefill batch of the same model
        dict(name="route_groups_32768", **_route(32768, 256, 8, "sigmoid", True, 8, 4, 2, True, 2.5, "f32")),
        # one token of a decode step, the row for the router and the 8-bit one for the experts
        dict(name="norm_decode_1", **_norm(1, 2048, "bf16", True, True, True)),
        # a ragged chunk in f16, hidden size no power of two, no 8-bit form
        dict(name="norm_f16_1000", **_norm(1000, 2880, "f16", True, True, False)),
        # a large ragged prefill batch with the 8-bit form
        dict(name="norm_8191", **_norm(8191, 4096, "bf16", True, True, True)),
        # single-user decode: a few experts' weights, cold
        dict(name="moe_q30b_decode_1", **_moe(Q30B, 1, "bf16")),
        # a small decode batch: every expert's weights once
        dict(name="moe_qwen3_decode_16", **_moe(QWEN3, 16, "bf16")),
        # the same from the 8-bit rows of the norm
        dict(name="moe_qwen3_decode_8_rows8", **_moe(QWEN3, 8, "bf16", "8")),
        # an embedding model in f16, a ragged batch of short documents
        dict(name="moe_embed_f16_777", **_moe(EMBED, 777, "f16")),
        # a prefill chunk over many small experts
        dict(name="moe_q30b_prefill_4096", **_moe(Q30B, 4096, "bf16")),
        # the largest prefill batch, from 8-bit rows
        dict(name="moe_qwen3_prefill_16384_rows8", **_moe(QWEN3, 16384, "bf16", "8")),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(2 ** rng.uniform(math.log2(lo), math.log2(hi))))))


def draw(rng):
    kind = rng.choice(["route", "norm", "moe", "moe", "moe"])
    if kind == "route":
        E = rng.choice([8, 16, 32, 60, 64, 128, 160, 256, 384, 512])
        T = min(_log_int(rng, 1, 32768), 32768 * 256 // E)
        groups = rng.choice([g for g in (1, 1, 2, 4, 8) if E % g == 0 and E // g >= 4])
        topk_groups = rng.randint(max(1, groups // 2), groups)
        k = rng.randint(1, min(8, topk_groups * (E // groups)))
        score = rng.choice(["softmax", "sigmoid"])
        return _route(T, E, k, score, rng.random() < 0.5, groups, topk_groups, rng.randint(1, 2),
                      rng.random() < 0.7, rng.choice([1.0, 2.5]), rng.choice(["f32", "f32", "bf16", "f16"]))
    if kind == "norm":
        H = 32 * _log_int(rng, 8, 256)
        T = min(_log_int(rng, 1, 32768), 8191 * 4096 // H)
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        wide, mx = rng.choice([(True, True), (True, False), (False, True)])
        return _norm(T if dtype != "f32" else max(1, T // 2), H, dtype, rng.random() < 0.7, wide, mx)
    model = rng.choice([QWEN3, Q30B, EMBED, None, None])
    if model is None:
        E = rng.choice([4, 8, 16, 32, 60, 64])
        model = dict(H=32 * _log_int(rng, 8, 128), I=32 * _log_int(rng, 8, 64), E=E, k=rng.randint(1, min(8, E)),
                     act=rng.choice(["silu", "gelu", "relu"]), moe_type=rng.randint(0, 1))
    per_token = model["k"] * 2 * (3 if model["moe_type"] == 0 else 2) * model["H"] * model["I"]
    T = max(1, min(_log_int(rng, 1, 16384), int(1.2e12 / per_token)))
    return _moe(model, T, rng.choice(["bf16", "bf16", "f16"]), rng.choice(["16", "16", "8"]), rng.random() < 0.25,
                rng.random() < 0.25)


# ------------------------------------------------------------------- inputs
def _normal(shape, dtype, gen, std=1.0):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=gen)


def _exponents(amax, largest):
    """The least e with amax <= largest * 2^e, as the byte e + 127 (0 for a block of zeros)."""
    m, e = torch.frexp(amax / largest)  # amax / largest = m 2^e, 0.5 <= m < 1
    e = torch.where(m == 0.5, e - 1, e)
    return torch.where(amax > 0, (e + 127).clamp(0, 254), torch.zeros_like(e)).to(torch.uint8)


def _mxfp4(w):
    """codes [.., K/2] (k even in the low nibble) and scale bytes [.., K/32] of w [.., K] f32."""
    b = w.unflatten(-1, (-1, 32))
    s = _exponents(b.abs().amax(-1), 6.0)
    v = b * torch.exp2(127.0 - s.float()).unsqueeze(-1)
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=w.device)
    # a tie goes to the even code: edges 0.25, 1.25, 2.5, 5 round down, the others up
    a = v.abs()
    c = (a.unsqueeze(-1) > edges).sum(-1, dtype=torch.uint8)
    c += ((a == 0.75) | (a == 1.75) | (a == 3.5)).to(torch.uint8)
    c |= (v < 0).to(torch.uint8) << 3
    c = c.flatten(-2).unflatten(-1, (-1, 2))
    return c[..., 0] | (c[..., 1] << 4), s


def _mxfp4_experts(E, N, K, gen):
    codes = torch.empty((E, N, K // 2), dtype=torch.uint8, device="cuda")
    scales = torch.empty((E, N, K // 32), dtype=torch.uint8, device="cuda")
    per = max(1, (1 << 25) // (N * K))
    for e in range(0, E, per):
        n = min(per, E - e)
        codes[e:e + n], scales[e:e + n] = _mxfp4(_normal((n, N, K), torch.float32, gen, 0.02))
    return codes, scales


def _mxfp8(y):
    """codes [.., K] (float8_e4m3fn) and scale bytes [.., K/32] of y [.., K] f32."""
    b = y.unflatten(-1, (-1, 32))
    s = _exponents(b.abs().amax(-1), 448.0)
    v = b * torch.exp2(127.0 - s.float()).unsqueeze(-1)
    return v.flatten(-2).to(torch.float8_e4m3fn), s


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) * 7919 + 29)
    T, dt = case["T"], DTYPES[case["dtype"]]
    s = {"case": case}
    if case["kind"] == "route":
        E, k = case["E"], case["k"]
        s["logits"] = _normal((T, E), dt, gen)
        s["bias"] = _normal((E,), torch.float32, gen, 0.1) if case["bias"] else None
        s["w"] = torch.empty((T, k), dtype=torch.float32, device="cuda")
        s["i"] = torch.empty((T, k), dtype=torch.int32, device="cuda")
        s["ei"] = torch.empty((T, k), dtype=torch.int32, device="cuda")
        return s
    if case["kind"] == "norm":
        H = case["H"]
        # rows of different loudness, as a residual stream has
        loud = torch.exp2(_normal((T, 1), torch.float32, gen))
        s["x"] = (_normal((T, H), torch.float32, gen) * loud).to(dt)
        s["residual"] = (_normal((T, H), torch.float32, gen) * loud * 2).to(dt) if case["residual"] else None
        s["weight"] = (1 + _normal((H,), torch.float32, gen, 0.1)).to(dt)
        s["residual_out"] = torch.empty_like(s["x"]) if case["residual"] else None
        s["out"] = torch.empty_like(s["x"]) if case["wide"] else None
        s["codes"] = torch.empty((T, H), dtype=torch.uint8, device="cuda") if case["mx"] else None
        s["scales"] = torch.empty((T, H // 32), dtype=torch.uint8, device="cuda") if case["mx"] else None
        return s
    H, I, E, k = case["H"], case["I"], case["E"], case["k"]
    logits = _normal((T, E), torch.float32, gen)
    if case["skew"]:  # some experts are favoured, as trained routers do
        favour = 4.0 / (1.0 + torch.arange(E, device="cuda", dtype=torch.float32))
        logits += favour[torch.randperm(E, generator=gen, device="cuda")]
    p, idx = torch.softmax(logits, -1).topk(k, -1)
    s["rw"] = (p / p.sum(-1, keepdim=True)).contiguous()
    if case["dropped"]:  # the rows of a padded batch go to no expert, and some pairs of others
        gone = (torch.arange(T, device="cuda") >= T - T // 8).unsqueeze(1) | (
            torch.rand((T, k), generator=gen, device="cuda") < 0.05)
        idx = torch.where(gone, E, idx)
    s["idx"] = idx.to(torch.int32).contiguous()
    x = _normal((T, H), torch.float32, gen)
    if case["rows"] == "8":
        codes, s["x_scale"] = _mxfp8(x)
        s["x"] = codes.view(torch.uint8)
    else:
        s["x"], s["x_scale"] = x.to(dt), None
    s["gate"], s["gate_s"] = _mxfp4_experts(E, I, H, gen)
    s["up"], s["up_s"] = _mxfp4_experts(E, *((I, H) if case["moe_type"] == 0 else (H, I)), gen)
    s["down"], s["down_s"] = _mxfp4_experts(E, H, I, gen) if case["moe_type"] == 0 else (None, None)
    return s


# ------------------------------------------------------------- plain forms
def _pow2(s):
    return torch.exp2(s.float() - 127.0)


def _from_mxfp4(codes, scales):
    values = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    nib = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    return (values[nib.int()].unflatten(-1, (-1, 32)) * _pow2(scales).unsqueeze(-1)).flatten(-2)


def _act(x, act):
    if act == "silu":
        return x / (1 + torch.exp(-x))
    if act == "gelu":
        return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))
    return x.clamp_min(0)


def _plain_route(s):
    c, l = s["case"], s["logits"].double()
    T, k = c["T"], c["k"]
    if c["score"] == "softmax":
        e = torch.exp(l - l.amax(-1, keepdim=True))
        p = e / e.sum(-1, keepdim=True)
    else:
        p = 1 / (1 + torch.exp(-l))
    rank = p + s["bias"].double() if s["bias"] is not None else p
    g = rank.unflatten(-1, (c["groups"], -1))
    of_group = g.sort(dim=-1, descending=True).values[..., :c["group_top"]].sum(-1)
    order = of_group.sort(dim=-1, descending=True, stable=True).indices
    keep = torch.zeros_like(of_group).scatter_(-1, order[:, :c["topk_groups"]], 1.0) > 0
    rank = torch.where(keep.unsqueeze(-1), g, -math.inf).flatten(-2)
    idx = rank.sort(dim=-1, descending=True, stable=True).indices[:, :k]
    w = p.gather(-1, idx)
    if c["renorm"]:
        w = w / w.sum(-1, keepdim=True)
    t = torch.arange(T, device=idx.device, dtype=torch.int32).unsqueeze(1)
    j = torch.arange(k, device=idx.device, dtype=torch.int32)
    return {"w": (w * c["scale"]).float(), "i": idx.int(), "ei": j * T + t}


def _plain_norm(s):
    c, out = s["case"], {}
    x = s["x"].float()
    if s["residual"] is not None:
        x = x + s["residual"].float()
        out["residual"] = x.to(s["x"].dtype)
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s["weight"].float()
    if c["wide"]:
        out["y"] = y.to(s["x"].dtype)
    if c["mx"]:
        out["codes"], scales = _mxfp8(y)
        out["scales"] = scales.view(torch.float8_e8m0fnu)
    return out


def _plain_moe(s):
    c = s["case"]
    T, E, k, dt = c["T"], c["E"], c["k"], DTYPES[c["dtype"]]
    x = s["x"]
    if s["x_scale"] is not None:
        x = (x.view(torch.float8_e4m3fn).float().unflatten(-1, (-1, 32)) * _pow2(s["x_scale"]).unsqueeze(-1)).flatten(-2)
    x = x.float()
    idx = s["idx"].long().flatten()
    last = (s["down"], s["down_s"]) if c["moe_type"] == 0 else (s["up"], s["up_s"])
    first = [(s["gate"], s["gate_s"])] + ([(s["up"], s["up_s"])] if c["moe_type"] == 0 else [])
    if T * k < E or T * k <= 16:
        # few pairs: each with its expert's weights
        e = idx.clamp_max(E - 1)
        rows = x.repeat_interleave(k, 0).unsqueeze(1)
        which = lambda w: _from_mxfp4(w[0][e], w[1][e])  # noqa: E731
    else:
        # the pairs of each expert side by side, as many as the fullest has
        order = idx.sort(dim=0, stable=True).indices
        count = torch.bincount(idx, minlength=E + 1)
        place = torch.arange(T * k, device=idx.device) - (count.cumsum(0) - count)[idx[order]]
        most = int(count[:E].max().clamp_min(1))
        rows = x.new_zeros((E + 1, max(most, int(count[E])), x.shape[1]))
        rows[idx[order], place] = x[order // k]
        rows = rows[:E, :most]
        which = lambda w: _from_mxfp4(*w)  # noqa: E731
    h = [torch.matmul(rows, which(w).transpose(-1, -2)) for w in first]
    h = _act(h[0], c["act"]) * h[1] if len(h) == 2 else _act(h[0], c["act"])
    y = torch.matmul(h, which(last).transpose(-1, -2))
    if T * k < E or T * k <= 16:
        pairs = y.squeeze(1)
    else:
        pairs = y.new_zeros((T * k, y.shape[-1]))
        taken = idx[order] < E
        at = order[taken]
        pairs[at] = y[idx[at], place[taken]]
    w = torch.where(idx < E, s["rw"].flatten(), 0.0)
    return (pairs * w.unsqueeze(-1)).unflatten(0, (T, k)).sum(1).to(dt)


def run(state):
    s = state
    c = s["case"]
    if not own:
        return {"route": _plain_route, "norm": _plain_norm, "moe": _plain_moe}[c["kind"]](s)
    cm = _package()
    if c["kind"] == "route":
        cm.topk_route(s["logits"], s["w"], s["i"], s["ei"], bias=s["bias"], score=c["score"], num_groups=c["groups"],
                      topk_groups=c["topk_groups"], group_top=c["group_top"], renormalize=c["renorm"],
                      scale=c["scale"])
        return {"w": s["w"], "i": s["i"], "ei": s["ei"]}
    if c["kind"] == "norm":
        cm.add_rms_norm(s["x"], s["weight"], EPS, residual=s["residual"], residual_output=s["residual_out"],
                        output=s["out"], codes=s["codes"], scales=s["scales"])
        out = {}
        if s["residual"] is not None:
            out["residual"] = s["residual_out"]
        if c["wide"]:
            out["y"] = s["out"]
        if c["mx"]:
            out["codes"] = s["codes"].view(torch.float8_e4m3fn)
            out["scales"] = s["scales"].view(torch.float8_e8m0fnu)
        return out
    out = torch.empty((c["T"], c["H"]), dtype=DTYPES[c["dtype"]], device=s["x"].device)
    cm.fused_moe_mxfp4(s["x"], s["gate"], s["up"], s["down"], s["gate_s"], s["up_s"], s["down_s"], s["rw"], s["idx"],
                       out, c["E"], c["k"], activation=ACTS[c["act"]], moe_type=c["moe_type"],
                       input_scale=s["x_scale"], accumulate=False)
    return out


# ------------------------------------------------------------------- work
def work(case):
    T = case["T"]
    if case["kind"] == "route":
        E, k = case["E"], case["k"]
        return {"bytes": T * E * SIZE[case["dtype"]] + T * k * 12 + (4 * E if case["bias"] else 0), "flops": 4 * T * E}
    if case["kind"] == "norm":
        H, es = case["H"], SIZE[case["dtype"]]
        rows = (1 + 2 * case["residual"] + case["wide"]) * es + (1 + 1 / 32) * case["mx"]
        return {"bytes": T * H * rows + H * es, "flops": 6 * T * H}
    H, I, E, k = case["H"], case["I"], case["E"], case["k"]
    mats = 3 if case["moe_type"] == 0 else 2
    touched = E * (1 - (1 - k / E) ** T)  # of uniform routing
    x = 1 + 1 / 32 if case["rows"] == "8" else 2
    return {"bytes": touched * mats * H * I * (0.5 + 1 / 32) + T * H * (x + 2) + T * k * 8,
            "flops": 2 * mats * T * k * H * I}


# ---------------------------------------------- the definitions in 64 bits
def _exact_route(c, s):
    l = s["logits"].double().cpu().numpy()
    if c["score"] == "softmax":
        p = np.exp(l - l.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
    else:
        p = 1.0 / (1.0 + np.exp(-l))
    rank = p.copy()
    if s["bias"] is not None:
        rank += s["bias"].double().cpu().numpy()
    T, E, G = c["T"], c["E"], c["groups"]
    per = E // G
    groups = np.zeros((T, G))
    for g in range(G):
        best = np.sort(rank[:, g * per:(g + 1) * per], axis=1)
        groups[:, g] = best[:, per - 1] if c["group_top"] == 1 else best[:, per - 1] + best[:, per - 2]
    first = np.argsort(-groups, axis=1, kind="stable")[:, :c["topk_groups"]]
    allowed = np.zeros((T, G), dtype=bool)
    np.put_along_axis(allowed, first, True, axis=1)
    rank[~np.repeat(allowed, per, axis=1)] = LOWEST
    idx = np.argsort(-rank, axis=1, kind="stable")[:, :c["k"]]
    w = np.take_along_axis(p, idx, 1)
    if c["renorm"]:
        w /= w.sum(1, keepdims=True)
    ei = np.arange(c["k"])[None, :] * T + np.arange(T)[:, None]
    return {"w": w * c["scale"], "i": idx.astype(np.int64), "ei": ei.astype(np.int64)}


def _exact_norm(c, s):
    out = {}
    x = s["x"].double()
    if s["residual"] is not None:
        x = x + s["residual"].double()
        out["residual"] = x
    y = x / torch.sqrt(torch.mean(x.square(), dim=1, keepdim=True) + EPS) * s["weight"].double()
    if c["wide"]:
        out["y"] = y
    if c["mx"]:
        blocks = y.reshape(c["T"], -1, 32)
        most = blocks.abs().max(dim=2).values
        e = torch.ceil(torch.log2(most / 448.0))
        e = torch.where(torch.ldexp(torch.full_like(e, 448.0), e) < most, e + 1, e)  # log2's own rounding
        e = torch.where(torch.ldexp(torch.full_like(e, 448.0), e - 1) >= most, e - 1, e)
        e = torch.where(most > 0, e.clamp(-127, 127), torch.full_like(e, -127.0))
        v = torch.ldexp(blocks, -e.unsqueeze(2))
        # e4m3: steps of 2^(exponent - 3), of 2^-9 below 2^-6; ties to even
        step = torch.ldexp(torch.ones_like(v), torch.frexp(v).exponent.clamp_min(-5) - 4)
        out["codes"] = (torch.round(v / step) * step).reshape(c["T"], -1)
        out["scales"] = torch.ldexp(torch.ones_like(e), e)
    return out


def _exact_weights(codes, scales):
    sign = 1.0 - 2.0 * ((codes >> 3) & 1).double()
    exponent, mantissa = ((codes >> 1) & 3).double(), (codes & 1).double()
    v = torch.where(exponent == 0, 0.5 * mantissa, torch.exp2(exponent - 1) * (1 + 0.5 * mantissa)) * sign
    return v * torch.exp2(scales.double() - 127).repeat_interleave(32, dim=1)


def _exact_moe(c, s):
    x = s["x"]
    if s["x_scale"] is not None:
        x = x.view(torch.float8_e4m3fn).float().double() * torch.exp2(s["x_scale"].double() - 127).repeat_interleave(32, 1)
    x = x.double()
    out = torch.zeros((c["T"], c["H"]), dtype=torch.float64, device=x.device)

    def matrix(q, scale, e):
        low, high = q[e] & 15, q[e] >> 4
        both = torch.empty((q.shape[1], q.shape[2] * 2), dtype=torch.uint8, device=q.device)
        both[:, 0::2], both[:, 1::2] = low, high
        return _exact_weights(both, scale[e])

    for e in range(c["E"]):
        t, j = torch.where(s["idx"] == e)
        if t.numel() == 0:
            continue
        a = x[t] @ matrix(s["gate"], s["gate_s"], e).t()
        if c["act"] == "silu":
            a = a * torch.sigmoid(a)
        elif c["act"] == "gelu":
            a = a * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (a + 0.044715 * a ** 3))
        else:
            a = torch.relu(a)
        if c["moe_type"] == 0:
            a = a * (x[t] @ matrix(s["up"], s["up_s"], e).t())
            y = a @ matrix(s["down"], s["down_s"], e).t()
        else:
            y = a @ matrix(s["up"], s["up_s"], e).t()
        out.index_add_(0, t, y * s["rw"][t, j].double().unsqueeze(1))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"route": _exact_route, "norm": _exact_norm, "moe": _exact_moe}[case["kind"]](case, s)
