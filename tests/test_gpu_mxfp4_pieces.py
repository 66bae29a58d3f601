"""MXFP4 batches whose f32 pair rows would pass 2 GiB go in pieces over one workspace:
the same results, bounded memory, also captured."""
import pytest
import torch

import candle_moe as cm
import operator_reference as ref
from test_gpu_mxfp4 import BF, F16, run, setup

pytestmark = pytest.mark.gpu
H, I, E, k = 4096, 32, 16, 8  # a piece: 2^31 / (4 H k) = 16384 tokens


def check(s, out, before=None):
    x = s["x"] if s["x_scale"] is None else ref.from_mxfp8(s["x"], s["x_scale"])
    w = [ref.from_mxfp4(*q) if q[0] is not None else None for q in (s["gate"], s["up"], s["down"])]
    aligned = 2.0 ** -12 if s["x_scale"] is not None and s["dtype"] == BF else 0.0
    y, far = ref.moe(x, *w, s["rw"], s["idx"], 0, s["moe_type"], s["dtype"], rounded=False, aligned=aligned)
    if before is not None:
        y = y + before.double()
        far = far + ref.HALF[s["dtype"]] * (y.abs() + far)
    ref.within(out, y, far)


@pytest.mark.parametrize("T, moe_type, dtype, rows8", [(40000, 0, BF, False), (32769, 1, F16, True), (16385, 0, BF, True)])
def test_pieces(T, moe_type, dtype, rows8):
    s = setup(T, H, I, E, k, moe_type, dtype, rows8, seed=T, dropped=0.05)
    out = torch.full((T + 1, H), 3.0, dtype=dtype, device="cuda")
    cm.trim_workspaces()
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    run(s, 0, out[:T])
    torch.cuda.synchronize()
    # the rows of a piece (2 GiB), half as much to grow, and half a GiB for all else
    assert free - torch.cuda.mem_get_info()[0] <= 3.5 * 2 ** 30
    assert (out[T] == 3).all()
    check(s, out[:T])
    acc = torch.randn(T, H, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    before = acc.clone()
    run(s, 0, acc, accumulate=True)
    check(s, acc, before)


def test_captured():
    T = 20000
    s = setup(T, H, I, E, k, 0, BF, False, seed=3)
    few = setup(300, H, I, E, k, 0, BF, False, seed=4)
    outs = [torch.empty(n, H, dtype=BF, device="cuda") for n in (T, 300)]
    cm.trim_workspaces()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        run(s, 0, outs[0])
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in outs]
    for g, c, o in zip(graphs, (s, few), outs):
        with torch.cuda.graph(g, stream=st):
            run(c, 0, o)
    for _ in range(3):
        for g, c, o in zip(graphs, (s, few), outs):
            c["x"].copy_(c["x"].flip(0))
            eager = run(c, 0, torch.empty_like(o))
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(eager, o)
    check(few, outs[1])
