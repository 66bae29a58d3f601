"""The operators around the expert products in plain 64-bit form, from their
definitions, for the tests (torch, on whatever device the inputs are on)."""
import math

import numpy as np
import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # half a step, relative
LEAST = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}  # half the least step
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


# ------------------------------------------------------------------- routing
def route(logits, k, bias=None, score="softmax", num_groups=1, topk_groups=1, group_top=1, renormalize=True, scale=1.0):
    """(weights f64, indices, j * T + t) of numpy logits [T, E]."""
    l = np.asarray(logits, dtype=np.float64)
    T, E = l.shape
    with np.errstate(all="ignore"):
        if score == "softmax":
            m = np.fmax.reduce(l, axis=1, keepdims=True)
            p = np.where(l == -np.inf, 0.0, np.exp(l - m))
            total = p.sum(1, keepdims=True)
            p = np.where(total == 0.0, 0.0, p / total)
        else:
            p = 1.0 / (1.0 + np.exp(-l))
        c = p + (0.0 if bias is None else np.asarray(bias, np.float64))
        c = np.where(np.isnan(c), -np.inf, c)
        per = E // num_groups
        best = -np.sort(-c.reshape(T, num_groups, per), axis=2)
        g = best[:, :, 0] if group_top == 1 else best[:, :, 0] + best[:, :, 1]
        g = np.where(np.isnan(g), -np.inf, g)
        w, idx = np.zeros((T, k)), np.zeros((T, k), np.int64)
        for t in range(T):
            groups = sorted(range(num_groups), key=lambda q: (-g[t, q], q))[:topk_groups]
            experts = [e for q in groups for e in range(q * per, (q + 1) * per)]
            idx[t] = sorted(experts, key=lambda e: (-c[t, e], e))[:k]
            w[t] = p[t, idx[t]]
        if renormalize:
            total = w.sum(1, keepdims=True)
            w = np.where(total == 0.0, 0.0, w / total)
    ei = np.arange(k)[None, :] * T + np.arange(T)[:, None]
    return w * scale, idx, ei


# -------------------------------------------------------------------- formats
def mx_scale(amax, largest):
    """Scale bytes: the least e with amax <= largest * 2^e, + 127."""
    m, e = torch.frexp(amax.double() / largest)
    e = torch.where(m == 0.5, e - 1, e) + 127
    s = torch.where(amax > 0, e.clamp(0, 254), torch.zeros_like(e))
    return torch.where(torch.isfinite(amax), s, torch.full_like(s, 255)).to(torch.uint8)


def scale_value(s):
    v = torch.exp2(s.double() - 127)
    return torch.where(s == 255, torch.full_like(v, math.nan), v)


def mxfp4(w):
    """codes [.., K / 2], scales [.., K / 32] of w [.., K] (any float type)."""
    b = w.double().unflatten(-1, (-1, 32))
    s = mx_scale(b.abs().amax(-1), 6.0)
    v = torch.where((s == 255).unsqueeze(-1), torch.zeros_like(b), b / torch.exp2(s.double() - 127).unsqueeze(-1))
    values = torch.tensor(E2M1, dtype=torch.float64, device=w.device)
    far = (v.abs().unsqueeze(-1) - values).abs()
    # the nearest value; of two the one with the even code
    near = far == far.amin(-1, keepdim=True)
    order = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7], device=w.device)
    c = order[near[..., order].int().argmax(-1)].to(torch.uint8)
    c = (c | ((v < 0).to(torch.uint8) << 3)).flatten(-2).unflatten(-1, (-1, 2))
    return c[..., 0] | (c[..., 1] << 4), s


def from_mxfp4(codes, scales):
    values = torch.tensor(E2M1 + [-v for v in E2M1], dtype=torch.float64, device=codes.device)
    v = values[torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()]
    return (v.unflatten(-1, (-1, 32)) * scale_value(scales).unsqueeze(-1)).flatten(-2)


def from_mxfp8(codes, scales):
    v = codes.view(torch.float8_e4m3fn).to(torch.float32).double()
    return (v.unflatten(-1, (-1, 32)) * scale_value(scales).unsqueeze(-1)).flatten(-2)


# ----------------------------------------------------------------------- norm
def norm(x, weight, eps, residual=None):
    """(z, y) in 64 bits."""
    z = x.double() + (0.0 if residual is None else residual.double())
    return z, z / torch.sqrt(z.square().mean(-1, keepdim=True) + eps) * weight.double()


# ------------------------------------------------------------------------ MoE
def act64(x, act):
    if act == 0:
        return x * torch.sigmoid(x)
    if act == 1:
        return x * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3))
    return torch.relu(x)


def moe(x, gate, up, down, rw, idx, act, moe_type, dtype, rounded=True, aligned=0.0):
    """The MoE in 64 bits over weights [E, N, K], and how far a result of `dtype`
    may be from it: the intermediate, each pair's row and the output rounded to
    dtype once (half a step each), f32 sums (2^-24 per term and rounding), the
    activation within 2^-20 (its slope is at most 1.13). aligned: of the first
    products' sum of magnitudes, what their sums may lose (8-bit rows on the scaled
    matrix instruction, which aligns 64 terms to the largest: 64 * 2^-18 of it)."""
    T, H = x.shape
    E = gate.shape[0]
    u, tiny = HALF[dtype], LEAST[dtype]
    out = torch.zeros((T, H), dtype=torch.float64, device=x.device)
    far = torch.zeros_like(out)
    for e in range(E):
        t, j = torch.where(idx == e)
        if not t.numel():
            continue
        a, g = x[t].double(), gate[e].t()
        s, ds = a @ g, (a.abs() @ g.abs()) * ((a.shape[1] + 4) * 2.0 ** -24 + aligned)
        h, dh = act64(s, act), 1.13 * ds + 2.0 ** -20 * act64(s, act).abs() + 2.0 ** -126
        last = up[e].t()
        if moe_type == 0:
            v, dv = a @ last, (a.abs() @ last.abs()) * ((a.shape[1] + 4) * 2.0 ** -24 + aligned)
            dh = dh * (v.abs() + dv) + h.abs() * dv
            h = h * v
            last = down[e].t()
        dh = dh + u * (h.abs() + dh) + tiny
        y = h @ last
        dy = dh @ last.abs() + ((h.abs() + dh) @ last.abs()) * (h.shape[1] + 4) * 2.0 ** -24
        w = rw[t, j].double().unsqueeze(1)
        dy = w.abs() * (dy + 2.0 ** -22 * y.abs())
        if rounded:
            dy = dy + u * (w * y).abs() + tiny
        out.index_add_(0, t, w * y)
        far.index_add_(0, t, dy)
    return out, far * (1 + u) + u * out.abs() + tiny


def within(got, want, far, what=""):
    got = got.double()
    off = (got - want).abs()
    bad = ~(off <= far)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {got.numel()} values too far off, the worst "
                           f"{float((off / far).nan_to_num(float('inf')).max()):.3g} of what is allowed")
