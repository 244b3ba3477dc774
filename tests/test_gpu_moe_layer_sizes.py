"""The 4-bit mixture-of-experts layer at the sizes that its kernels differ in, with inputs at
any alignment, and without an allocation, against its definition in 64 bits."""
import numpy as np
import pytest
import torch

from moe_layer_cases import CASES, PART_CASES
from test_gpu_moe_layer import Layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", [c[1] for c in CASES], ids=["%d-%s" % (i, "-".join(str(v) for v in c[0]))
                                                             for i, c in enumerate(CASES)])
def test_sizes(hip, case):
    p = Layer(hip, **case)
    p.run()
    p.check()


@pytest.mark.parametrize("kx,kr", [("f32", "bf16"), ("bf16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("gap", [0, 1])
def test_any_alignment(hip, kx, kr, gap):
    """Rows of x, the router and the output that start at any element."""
    p = Layer(hip, t=5, embd=264, ff=48, kx=kx, ky=kx, kr=kr, x_gap=gap, y_gap=gap)
    whole = {}
    for name in ("x", "router"):
        a = p.d[name].reshape(-1)
        whole[name] = torch.zeros(a.numel() + 1, dtype=a.dtype, device="cuda")
        whole[name][1:] = a
        p.d[name] = whole[name][1:]
    p.layer.router = p.d["router"].data_ptr()
    buf = torch.full((p.out.numel() + 2,), 77.0, dtype=p.out.dtype, device="cuda")
    p.out = buf[1:-1].view(p.out.shape)
    p.run()
    p.check()
    assert buf[0] == 77.0 and buf[-1] == 77.0


def test_the_workspace_is_enough(hip):
    """Nothing is written behind the workspace, the ids or the weights; nothing is allocated."""
    for case in (dict(t=1, embd=1, ff=1, experts=1, k=1), dict(t=32, embd=129, ff=127, experts=9, k=9, shared=2),
                 dict(t=7, embd=600, ff=40, experts=300, k=5, ky="bf16")):
        p = Layer(hip, **case)
        n = p.work.numel()
        room = torch.full((n + 512,), 0xCD, dtype=torch.uint8, device="cuda")
        p.work = room[:n]
        for name in ("ids", "weights"):
            a = getattr(p, name)
            more = torch.full((a.numel() + 4,), 99, dtype=a.dtype, device="cuda")
            setattr(p, "more_" + name, more)
            setattr(p, name, more[:a.numel()].view(a.shape))
        before = hip.device_allocations()
        p.run()
        assert hip.device_allocations() == before
        p.check()
        assert (room[n:] == 0xCD).all()
        assert (p.more_ids[-4:] == 99).all() and (p.more_weights[-4:] == 99).all()


def test_a_token_alone_and_among_others(hip):
    """What a token gets does not depend on the tokens beside it, but for the order in which
    its experts' parts are added."""
    p = Layer(hip, t=32, embd=384, ff=160, experts=16, k=4, score=1, bias=True)
    p.run()
    p.check()
    ids, weights, out = p.ids.clone(), p.weights.clone(), p.out.clone()
    _, _, _, tol = p.want()
    for t in (0, 13, 31):
        one = Layer(hip, t=1, embd=384, ff=160, experts=16, k=4, score=1, bias=True)
        one.m, one.router, one.router_t, one.bias = p.m, p.router, p.router_t, p.bias
        one.x, one.xt = p.x[t:t + 1], p.xt[t:t + 1]
        one.upload()
        one.run()
        one.check()
        assert torch.equal(one.ids[0], ids[t]) and torch.equal(one.weights[0], weights[t])
        # (both are within tol of the same value)
        assert (np.abs((one.out[0] - out[t]).cpu().double().numpy()) <= 2 * tol[t]).all()


@pytest.mark.parametrize("case", PART_CASES, ids=lambda c: "-".join(str(c[n]) for n in ("t", "embd", "ff", "experts", "k")))
def test_down_products_in_parts(hip, case):
    """Eager, then captured and replayed: the same bits, a token that is not finite among them."""
    p = Layer(hip, **case)
    p.x[2, 0] = np.nan
    p.xt = torch.from_numpy(p.x).to(p.xt.dtype)
    p.upload()
    room = torch.full((p.work.numel() + 512,), 0xCD, dtype=torch.uint8, device="cuda")
    p.work = room[:-512]
    p.run()
    p.check()
    assert (room[-512:] == 0xCD).all()
    want = p.out.clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        p.run()
    for _ in range(3):
        p.out.fill_(77.0)
        p.work.random_(0, 256)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(torch.nan_to_num(p.out), torch.nan_to_num(want))
