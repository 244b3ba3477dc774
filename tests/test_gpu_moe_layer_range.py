"""The 4-bit mixture-of-experts layer at the ends of its types' ranges: the largest and the
smallest numbers in x and in h, weights of every scale, against its definition in 64 bits."""
import numpy as np
import pytest
import torch

import mxfp4_ref as M
import serving_ref as R
from test_gpu_moe_layer import Layer

pytestmark = pytest.mark.gpu

FLT_MAX = float(np.finfo(np.float32).max)
#: what rounds to bf16's infinity from here on
NO_BF16 = 255.5 * 2.0 ** 120


def moe(p):
    """M.moe with a closer bound where a clamp holds a sum (its error is then nothing) and where
    silu has vanished: (ids, weights, out, how far out may be off)."""
    c = p.c
    p.want()
    gate, up, down = p.wide
    with np.errstate(all="ignore"):
        logits = np.stack([(row * p.router).sum(1) for row in p.x])
    bias = None if p.bias is None else p.bias.astype(np.float64)
    ids, weights = R.route(logits, bias, c["k"], c["groups"], c["top_groups"], c["group_top"], c["score"], c["renorm"],
                           c["scale"])
    y, err = np.zeros(p.x.shape), np.zeros(p.x.shape)
    d, f, top = c["embd"], c["ff"], c["clamp"] if c["clamp"] > 1e-6 else np.inf
    cut = 2.0 ** -24 if c["ky"] == "f32" else 2.0 ** -16
    # Small h: two roundings to f32, 2^-150 each, and half a step of the last term, bf16's 2^-133
    # over 2^15 of three terms (2^-149), over 2^7 of two (2^-141)
    least = 2.0 ** -148 if c["ky"] == "f32" else 2.0 ** -140
    for t, x in enumerate(p.x):
        slots = [(e, w) for e, w in zip(ids[t], weights[t]) if e >= 0 and np.float32(w) != 0]
        slots += [(c["experts"] + j, 1.0) for j in range(c["shared"])]
        total = np.zeros(d)
        for e, w in slots:
            g, u = gate[e] @ x, up[e] @ x
            step = (d / 32 + 40) * 2.0 ** -23
            eg, eu = step * (np.abs(gate[e]) @ np.abs(x)), step * (np.abs(up[e]) @ np.abs(x))
            es = np.where((g - eg >= top) | (g + eg <= -200.0), 1e-80, 1.1 * eg)
            eu = np.where(np.abs(u) - eu >= top, 0.0, eu)
            g, u = np.minimum(g, top), np.clip(u, -top, top)
            with np.errstate(over="ignore"):
                s = g / (1.0 + np.exp(-g))
            h = s * u
            eh = es * (np.abs(u) + eu) + np.abs(s) * eu + np.abs(h) * (2.0 ** -20 + cut)
            y[t] += w * (down[e] @ h)
            err[t] += w * (np.abs(down[e]) @ eh) + least * np.abs(down[e]).sum(1)
            total += w * (np.abs(down[e]) @ np.abs(h))
        err[t] += (len(slots) * f / 32 + 40) * 2.0 ** -23 * total
    return ids, weights, y, err + M.rounding(y, c["ky"])


def check(p):
    p.run()
    want_ids, want_w, want, tol = moe(p)
    got = p.out[:, :p.c["embd"]].cpu().double().numpy()
    assert np.array_equal(p.ids.cpu().numpy(), want_ids)
    got_w = p.weights.cpu().double().numpy()
    assert (np.abs(got_w - want_w) <= np.abs(want_w) * (2.0 ** -24 + 2.0 ** -45) + 2.0 ** -150).all()
    assert np.isfinite(want).all() and np.isfinite(tol).all()
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (bad.sum(), np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], tol[bad][:5])


def scales(p, name, low, high, seed=1):
    rng = np.random.default_rng(seed)
    s = p.m[name][1]
    blocks = ((p.c["ff"] if name == "down" else p.c["embd"]) + 31) // 32
    s[:, :blocks] = rng.integers(low, high + 1, (len(s), blocks))


def tokens(p, x):
    p.xt, p.x = R.as_type(x, p.c["kx"])


#: f32 numbers that round to bf16's infinity, and the largest one that does not
TOP = [FLT_MAX, -FLT_MAX, NO_BF16, -NO_BF16, float(np.nextafter(np.float32(NO_BF16), np.float32(0)))]


@pytest.mark.parametrize("t,embd,ff", [(5, 256, 128), (5, 130, 64), (1, 4096, 96), (5, 4200, 40), (5, 8300, 33)])
@pytest.mark.parametrize("ky", ["f32", "bf16"])
def test_largest_x(hip, t, embd, ff, ky):
    """A finite x gives a finite row where the clamp holds what it makes of the sums: every
    weight is less than 1, so that the sums are finite in f32, too."""
    p = Layer(hip, t=t, embd=embd, ff=ff, clamp=7.0, shared=1, ky=ky, score=2)
    for name in ("gate", "up"):
        scales(p, name, 118, 124)
    x = p.x.copy()
    for i in range(t):
        x[i, [3, embd - 1][i % 2]] = TOP[i]
    tokens(p, x)
    p.upload()
    check(p)


def test_x_that_overflows_the_sums(hip):
    """Sums beyond f32's range, of one large term each: the clamp holds them; silu of such a
    sum below 0 is 0."""
    p = Layer(hip, t=5, embd=320, ff=64, clamp=10.0)
    for name in ("gate", "up"):
        scales(p, name, 128, 130)
    x = p.x.copy()
    for i in range(5):
        x[i, 7] = TOP[i]
    tokens(p, x)
    p.upload()
    check(p)


@pytest.mark.parametrize("t", [1, 3, 9])
@pytest.mark.parametrize("ky", ["f32", "bf16"])
def test_largest_h(hip, t, ky):
    """h between bf16's largest number and f32's: finite outputs where the down weights are small."""
    p = Layer(hip, t=t, embd=64, ff=128, experts=2, k=1, ky=ky)
    for name, s in (("gate", 127 + 64), ("up", 127 + 63)):
        codes, sc = p.m[name]
        codes[:], sc[:] = 0, 127
        # element 0 alone, 1 2^64 and +-1 2^63: h = +-x0^2 2^127
        codes[:, 0] = 2
        sc[:, 0] = s
    p.m["up"][0][::3, 0] = 10
    scales(p, "down", 100, 104)
    x = p.x.copy()
    x[:, 0] = np.sqrt(np.linspace(1.9975, 1.9999, t))
    tokens(p, x)
    p.upload()
    h = p.x[:, 0] ** 2 * 2.0 ** 127
    assert (h > NO_BF16).all() and (h < FLT_MAX).all()
    check(p)


#: exponent of x, scales of gate and up, of down
ENDS = {
    "tiny x, large weights": (-126, (250, 252), (116, 120)),
    "tiny x, the largest weights": (-127, (250, 254), (116, 120)),
    "large x, the smallest weights": (118, (0, 4), (116, 120)),
    "tiny h, large weights": (0, (58, 60), (248, 252)),
    "tiny h, the largest weights": (0, (58, 61), (250, 254)),
    "large h, the smallest weights": (0, (170, 172), (0, 4)),
}


@pytest.mark.parametrize("name", ENDS)
@pytest.mark.parametrize("kx,ky", [("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("t,embd,ff", [(1, 256, 128), (9, 300, 200), (3, 4500, 48), (2, 8300, 40), (4, 64, 1100)])
def test_scales_of_every_size(hip, name, kx, ky, t, embd, ff):
    """Weights of every scale against x or h that bring the sums back to ordinary sizes."""
    power, gate_up, down = ENDS[name]
    p = Layer(hip, t=t, embd=embd, ff=ff, kx=kx, ky=ky, experts=4, shared=1)
    scales(p, "gate", *gate_up)
    scales(p, "up", *gate_up, seed=2)
    scales(p, "down", *down, seed=3)
    tokens(p, p.x * 2.0 ** power)
    p.upload()
    check(p)


@pytest.mark.parametrize("t", [1, 6])
def test_largest_weights_and_f16_x(hip, t):
    """f16 x has no small numbers to bring such sums back: the clamp does."""
    p = Layer(hip, t=t, embd=200, ff=72, kx="f16", ky="f16", clamp=5.0)
    scales(p, "gate", 240, 254)
    scales(p, "up", 240, 254, seed=2)
    x = np.zeros_like(p.x)
    x[:, 5::64] = p.x[:, 5::64] * 2.0 ** -12
    tokens(p, x)
    p.upload()
    check(p)


@pytest.mark.parametrize("t,embd,ff", [(1, 256, 96), (7, 300, 130), (3, 4200, 40), (2, 8300, 33)])
@pytest.mark.parametrize("kx", ["f32", "bf16"])
def test_sums_that_leave_f32_on_the_way(hip, t, embd, ff, kx):
    """Terms of both signs beyond f32's range: what the clamp makes of their sum is finite."""
    p = Layer(hip, t=t, embd=embd, ff=ff, kx=kx, clamp=6.0, shared=1)
    for name in ("gate", "up"):
        scales(p, name, 126, 130, seed=ff)
    tokens(p, p.x * 5e37)
    p.upload()
    check(p)


@pytest.mark.parametrize("t,embd", [(1, 64), (32, 64), (9, 4400)])
def test_down_sums_that_leave_f32_on_the_way(hip, t, embd):
    """Two terms of h beyond f32's range that cancel; in parts (few rows) and whole."""
    p = Layer(hip, t=t, embd=embd, ff=1024, experts=2, k=1, ky="f32", clamp=8.0)
    for name in ("gate", "up"):  # rows 0 and 700 of every expert are the same: so is their h
        for a in p.m[name]:
            a.reshape(2, 1024, -1)[:, 700] = a.reshape(2, 1024, -1)[:, 0]
    codes, sc = p.m["down"]
    sc[:, 0], sc[:, 700 // 32] = 252, 252
    codes[:, 0], codes[:, 700 // 2] = 7, 15  # 6 and -6 2^125; nothing else in these bytes
    codes[:, 1:16], codes[:, 336:350], codes[:, 351:352] = 0, 0, 0
    x = p.x * 2.0 ** 20
    tokens(p, x)
    p.upload()
    _, _, want, _ = moe(p)
    p.run()
    got = p.out.cpu().double().numpy()
    # 1024 additions in 64 bits beside terms of 64 x 6 x 2^125
    assert (np.abs(got - want) <= 1024 * 2.0 ** -53 * 64 * 6 * 2.0 ** 125).all()


def test_nan_scales_stay_nan(hip):
    """Scales of 255 beside the largest ones: NaN, in the tokens that took that expert alone."""
    p = Layer(hip, t=6, experts=4, k=1, clamp=5.0)
    for name in ("gate", "up"):
        scales(p, name, 253, 254)
    p.m["gate"][1][2 * 128 + 5, 3] = 255
    tokens(p, p.x * 2.0 ** -127)
    p.upload()
    p.run()
    took = (p.ids.cpu().numpy() == 2).any(1)
    assert np.array_equal(np.isnan(p.out.cpu().numpy()).all(1), took)


@pytest.mark.parametrize("t,embd,ff", [(1, 256, 96), (6, 300, 130), (32, 64, 1100), (9, 5000, 40)])
def test_replayed_with_large_and_ordinary_x(hip, t, embd, ff):
    """Recorded once, replayed with x that leaves f32 on the way and with x that does not, in
    turn: every replay gives the eager run's bits, and the value."""
    p = Layer(hip, t=t, embd=embd, ff=ff, clamp=6.0, shared=1)
    for name in ("gate", "up"):
        scales(p, name, 126, 130, seed=ff)
    p.upload()
    x = p.x.copy()
    p.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p.run()
    for power in (5e37, 1.0, -5e37, 0.25):
        tokens(p, x * power)
        p.d["x"].copy_(p.xt.reshape(p.d["x"].shape))
        p.out.fill_(77.0)
        p.work.random_(0, 256)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        first = [a.clone() for a in (p.out, p.ids, p.weights)]
        check(p)
        assert all(torch.equal(a, b) for a, b in zip(first, (p.out, p.ids, p.weights)))
