"""A whole mixture-of-experts layer with 4-bit experts on the GPU, against its
definition in 64 bits."""
import numpy as np
import pytest
import torch

import mxfp4_ref as M
import serving_ref as R
from test_gpu_mxfp4 import dev, rows, stream

pytestmark = pytest.mark.gpu

BASE = dict(t=3, embd=256, ff=128, experts=8, shared=0, k=2, groups=1, top_groups=1, group_top=1, score=0, bias=False,
            renorm=True, scale=1.0, clamp=0.0, kx="f32", ky="f32", kr="f32", x_gap=0, y_gap=0)


class Layer:
    def __init__(self, hip, seed=0, router=None, biases=None, **kw):
        c = {**BASE, **kw}
        assert not set(kw) - set(BASE)
        self.hip, self.c = hip, c
        rng = np.random.default_rng(seed + c["t"] + 31 * c["embd"] + 7 * c["ff"])
        d, f, n, all_ = c["embd"], c["ff"], c["experts"], c["experts"] + c["shared"]
        at = 126 - int(np.log2(np.sqrt(d)) + 0.5)
        self.m = {"gate": M.random_rows(rng, all_ * f, d, at - 2, at), "up": M.random_rows(rng, all_ * f, d, at - 2, at)}
        at = 126 - int(np.log2(np.sqrt(f)) + 0.5)
        self.m["down"] = M.random_rows(rng, all_ * d, f, at - 2, at)
        self.router_t, self.router = R.as_type(rng.normal(0, 1.5, (n, d)) / np.sqrt(d) if router is None else router,
                                               c["kr"])
        self.bias = biases if biases is not None else rng.normal(0, 0.1, n).astype(np.float32) if c["bias"] else None
        self.xt, self.x = R.as_type(rng.normal(0, 1, (c["t"], d)), c["kx"])
        self.upload()

    def upload(self):
        c, hip, m = self.c, self.hip, self.m
        t, d = c["t"], c["embd"]
        self.d = {k: (dev(v[0]), dev(v[1])) for k, v in m.items()}
        self.d["router"] = dev(self.router_t)
        self.d["bias"] = dev(self.bias) if self.bias is not None else None
        self.d["x"], self.span = rows(self.xt, d + c["x_gap"])
        g, u, w = self.d["gate"], self.d["up"], self.d["down"]
        self.layer = hip.MoeMxfp4(
            router=self.d["router"].data_ptr(), router_len=self.d["router"].numel(), dtype_router=R.GGML[c["kr"]],
            bias=self.d["bias"].data_ptr() if self.bias is not None else 0,
            bias_len=c["experts"] if self.bias is not None else 0, gate=g[0].data_ptr(), up=u[0].data_ptr(),
            gate_up_len=g[0].numel(), gate_scales=g[1].data_ptr(), up_scales=u[1].data_ptr(),
            gate_up_scales_len=g[1].numel(), down=w[0].data_ptr(), down_len=w[0].numel(), down_scales=w[1].data_ptr(),
            down_scales_len=w[1].numel(), n_embd=d, n_ff=c["ff"], n_expert=c["experts"], n_shared=c["shared"],
            k=c["k"], n_group=c["groups"], topk_group=c["top_groups"], group_top=c["group_top"], score=c["score"],
            renormalise=int(c["renorm"]), scale=c["scale"], clamp=c["clamp"])
        self.out = torch.full((t, d + c["y_gap"]), 77.0, dtype=R.TORCH[c["ky"]], device="cuda")
        self.ids = torch.full((t, c["k"]), 99, dtype=torch.int32, device="cuda")
        self.weights = torch.full((t, c["k"]), 77.0, device="cuda")
        self.work = torch.full((max(1, hip.moe_mxfp4_work_bytes(self.layer, t)),), 0xCD, dtype=torch.uint8, device="cuda")

    def run(self):
        c, t, d = self.c, self.c["t"], self.c["embd"]
        self.hip.moe_mxfp4_dev(self.layer, self.out.data_ptr(), (t - 1) * (d + c["y_gap"]) + d, d + c["y_gap"],
                               self.ids.data_ptr(), self.weights.data_ptr(), self.ids.numel(), self.d["x"].data_ptr(),
                               self.span, d + c["x_gap"], self.work.data_ptr(), self.work.numel(), t, R.GGML[c["kx"]],
                               R.GGML[c["ky"]], stream())

    def want(self):
        c = self.c
        d, f, all_ = c["embd"], c["ff"], c["experts"] + c["shared"]
        if not hasattr(self, "wide"):
            v = {k: M.values(*m, f if k == "down" else d) for k, m in self.m.items()}
            self.wide = [v[k].reshape(all_, d if k == "down" else f, -1) for k in ("gate", "up", "down")]
        bias = None if self.bias is None else self.bias.astype(np.float64)
        return M.moe(self.x, self.router, bias, *self.wide, c["experts"], c["shared"], c["k"], c["groups"],
                     c["top_groups"], c["group_top"], c["score"], c["renorm"], c["scale"], c["clamp"], c["ky"])

    def check(self, ids=None):
        want_ids, want_w, want, tol = self.want()
        got_ids, got_w = self.ids.cpu().numpy(), self.weights.cpu().double().numpy()
        got = self.out[:, :self.c["embd"]].cpu().double().numpy()
        assert np.array_equal(got_ids, want_ids if ids is None else ids)
        # 64 bits rounded once, beside some 2^-48 of the scores
        assert (np.abs(got_w - want_w) <= np.abs(want_w) * (2.0 ** -24 + 2.0 ** -45) + 2.0 ** -150).all()
        assert np.array_equal(np.isnan(got), np.isnan(want))
        bad = ~(np.abs(got - want) <= tol) & ~np.isnan(want)
        assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], tol[bad][:5])
        assert (self.out[:, self.c["embd"]:] == 77.0).all()


CASES = [
    dict(t=1),
    dict(t=1, embd=1, ff=1, experts=1, k=1),
    dict(t=2, embd=32, ff=16, experts=3, k=3, renorm=False),
    dict(t=5, embd=33, ff=31, experts=5, k=1, score=1),
    dict(t=4, embd=129, ff=130, experts=16, k=4, score=2, bias=True, scale=1.5, clamp=10.0, shared=1),
    dict(t=7, embd=300, ff=200, experts=12, k=5, kx="bf16", ky="bf16", kr="bf16", x_gap=4, y_gap=8),
    dict(t=8, embd=520, ff=96, experts=64, k=8, kx="f16", ky="f16", kr="f16", x_gap=3, y_gap=1),
    dict(t=16, embd=1000, ff=352, experts=32, k=4, groups=4, top_groups=2, group_top=2, score=1, bias=True, scale=2.5,
         kx="f16", ky="f32"),
    dict(t=32, embd=256, ff=256, experts=8, k=2, kx="bf16", ky="f32", shared=2),
    dict(t=32, embd=200, ff=136, experts=4, k=4, ky="f16", clamp=0.5),
    dict(t=31, embd=384, ff=64, experts=256, k=6, score=2, bias=True, scale=1.5, clamp=10.0, shared=1),
    dict(t=9, embd=128, ff=128, experts=1024, k=32, score=0, renorm=False, kx="f32", ky="bf16"),
    dict(t=6, embd=640, ff=33, experts=100, k=10, groups=4, top_groups=1, group_top=1, score=0, shared=8),
    dict(t=17, embd=136, ff=520, experts=20, k=3, groups=5, top_groups=2, group_top=2, score=1, kx="bf16", ky="f16"),
    dict(t=3, embd=2048, ff=1024, experts=4, k=2, clamp=7.0),
    dict(t=12, embd=160, ff=160, experts=2, k=1, shared=1, kx="f32", ky="f32"),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join("%s%s" % i for i in c.items() if i[0] in ("t", "embd", "ff", "experts", "k")))
def test_layer(hip, case):
    p = Layer(hip, **case)
    p.run()
    p.check()


@pytest.mark.parametrize("t", [1, 4, 11, 32])
def test_equal_experts_go_by_id(hip, t):
    """Experts of the same router row are equal: the lower ids are chosen first."""
    rng = np.random.default_rng(5)
    row = rng.normal(0, 1, (1, 256)) / 16
    p = Layer(hip, t=t, experts=70, k=5, router=np.repeat(row, 70, 0))
    p.run()
    p.check(np.tile(np.arange(5, dtype=np.int32), (t, 1)))


@pytest.mark.parametrize("kx", ["f32", "bf16"])
def test_not_finite_tokens(hip, kx):
    """A NaN or an infinity in x: that token's row is NaN, the others are themselves."""
    p = Layer(hip, t=6, embd=300, kx=kx, shared=1, y_gap=4, score=1)
    p.x[1, 17], p.x[3, 299], p.x[4, 0] = np.nan, np.inf, -np.inf
    p.xt = torch.from_numpy(p.x).to(R.TORCH[kx])
    p.upload()
    p.run()
    p.check()


def test_tokens_without_experts(hip):
    """Biases of -inf leave experts out; with none left only the shared ones count."""
    for shared in (0, 1):
        for live in (0, 1, 3):
            bias = np.full(16, -np.inf, np.float32)
            bias[[9, 2, 14][:live]] = 0.0
            p = Layer(hip, t=5, experts=16, k=4, shared=shared, biases=bias, renorm=live != 1)
            p.run()
            assert (p.ids.cpu().numpy() >= 0).sum() == 5 * live
            p.check()


def test_experts_of_weight_zero_are_skipped(hip):
    """A scale of 0: routed experts count for nothing, even ones with NaN weights."""
    p = Layer(hip, t=4, scale=0.0, shared=1)
    for k in ("gate", "up", "down"):
        rows_ = 8 * (128 if k != "down" else 256)
        p.m[k][1][:rows_] = 255
    p.upload()
    p.run()
    p.check()


def test_nan_weights_stay_with_their_tokens(hip):
    """NaN blocks of one expert reach the tokens that chose it, and no other."""
    p = Layer(hip, t=9, experts=6, k=2)
    p.m["up"][1][3 * 128 + 5, 1] = 255
    p.upload()
    p.run()
    took = (p.ids.cpu().numpy() == 3).any(1)
    assert took.any() and not took.all()
    assert np.array_equal(np.isnan(p.out.cpu().numpy()).all(1), took)
    p.check()


@pytest.mark.parametrize("score", [0, 1, 2])
def test_large_logits(hip, score):
    """Scores at the ends of their ranges: softmax of far logits, sigmoids of 0 and 1."""
    rng = np.random.default_rng(8)
    p = Layer(hip, t=4, experts=12, k=3, score=score, router=rng.normal(0, 30, (12, 256)))
    p.run()
    p.check()


@pytest.mark.parametrize("case", [CASES[0], CASES[4], CASES[6], CASES[10]], ids=["t1", "t4", "t8", "t31"])
def test_graphs_and_streams(hip, case):
    """Captured and replayed with new tokens, on another stream, with a workspace that
    holds anything: every run is the eager one, bit for bit."""
    p = Layer(hip, **case)
    p.run()
    p.check()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        p.run()
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    for i in range(4):
        p.d["x"].copy_(torch.randn(p.d["x"].shape, device="cuda", generator=g))
        outs = []
        for how in ("graph", "eager", "stream"):
            for o in (p.out, p.ids, p.weights):
                o.fill_(55)
            p.work.random_(0, 256)
            torch.cuda.synchronize()
            if how == "graph":
                graph.replay()
            elif how == "eager":
                p.run()
            else:
                side = torch.cuda.Stream()
                with torch.cuda.stream(side):
                    p.run()
                side.synchronize()
            torch.cuda.synchronize()
            outs.append([o.clone() for o in (p.out[:, :p.c["embd"]], p.ids, p.weights)])
        for other in outs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(outs[0], other))


def test_two_streams_at_once(hip):
    """Two layers run at once on two streams, each with its own workspace."""
    ps = [Layer(hip, seed=s, **case) for s, case in enumerate((CASES[4], CASES[9], CASES[13]))]
    streams = [torch.cuda.Stream() for _ in ps]
    torch.cuda.synchronize()
    for _ in range(20):
        for p, s in zip(ps, streams):
            with torch.cuda.stream(s):
                p.run()
    torch.cuda.synchronize()
    for p in ps:
        p.check()


def test_experts_beyond_32_bit_offsets(hip):
    """Stacked experts of more than 2^32 bytes: the last as the first."""
    d, f, n = 8192, 4096, 280
    assert n * f * M.row_bytes(d) > 1 << 32
    p = Layer(hip, t=2, embd=d, ff=f, experts=2, k=1)
    small = [p.d[k] for k in ("gate", "up", "down")]
    big = [tuple(a.view(2, -1).repeat(n // 2, 1).reshape(-1) for a in m) for m in small]
    router = torch.zeros(n, d, device="cuda")
    router[n - 2:] = p.d["router"]  # the last two: the others' logits are 0
    bias = torch.full((n,), -10.0, device="cuda")
    bias[n - 2:] = 0.0
    p.run()
    first = [o.clone() for o in (p.out, p.ids, p.weights)]
    g, u, w = big
    layer = hip.MoeMxfp4(
        router=router.data_ptr(), router_len=router.numel(), bias=bias.data_ptr(), bias_len=n, gate=g[0].data_ptr(),
        up=u[0].data_ptr(), gate_up_len=g[0].numel(), gate_scales=g[1].data_ptr(), up_scales=u[1].data_ptr(),
        gate_up_scales_len=g[1].numel(), down=w[0].data_ptr(), down_len=w[0].numel(), down_scales=w[1].data_ptr(),
        down_scales_len=w[1].numel(), n_embd=d, n_ff=f, n_expert=n, n_shared=0, k=1, n_group=1, topk_group=1,
        group_top=1, score=2, renormalise=1, scale=1.0, clamp=0.0)
    work = torch.empty(hip.moe_mxfp4_work_bytes(layer, 2), dtype=torch.uint8, device="cuda")
    hip.moe_mxfp4_dev(layer, p.out.data_ptr(), p.out.numel(), d, p.ids.data_ptr(), p.weights.data_ptr(), 2,
                      p.d["x"].data_ptr(), p.span, d, work.data_ptr(), work.numel(), 2, 0, 0, stream())
    # (one expert of weight 1 whatever its score)
    assert torch.equal(p.ids, first[1] + n - 2) and torch.equal(p.weights, first[2]) and torch.equal(p.out, first[0])
