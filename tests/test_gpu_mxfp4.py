"""Microscaled 4-bit rows on the GPU: quantising and decoding bit for bit, the product
against 64-bit sums of the values that the codes stand for."""
import numpy as np
import pytest
import torch

import mxfp4_ref as M
import serving_ref as R

pytestmark = pytest.mark.gpu


def dev(a):
    return (a if isinstance(a, torch.Tensor) else torch.from_numpy(np.ascontiguousarray(a))).cuda()


def stream():
    return torch.cuda.current_stream().cuda_stream


def rows(t, stride):
    """t's rows on the GPU, `stride` apart and NaN between: (buffer, elements)."""
    buf, n = R.strided(t, stride)
    return dev(buf), n


def run_quantize(hip, t, kind, stride):
    n, k = t.shape
    x, span = rows(t, stride)
    codes = torch.full((n, M.row_bytes(k)), 0xAB, dtype=torch.uint8, device="cuda")
    scales = torch.full((n, M.scale_bytes(k)), 0xAB, dtype=torch.uint8, device="cuda")
    hip.quantize_mxfp4_dev(x.data_ptr(), span, stride, codes.data_ptr(), codes.numel(), scales.data_ptr(),
                           scales.numel(), n, k, R.GGML[kind], stream())
    return codes, scales


def hard_values(rng, n, k):
    """Rows with what a block can hold: borders between codes, zeros of both signs,
    blocks of nothing, the smallest and the largest numbers, wide ranges."""
    x = rng.normal(0, 1, (n, k)) * np.exp(rng.normal(0, 8, (n, 1)))
    for r in range(n):
        what = r % 8
        if what == 1:
            x[r] = rng.integers(-64, 65, k) / 8.0 * 2.0 ** rng.integers(-20, 20)
        elif what == 2:
            x[r] = np.where(rng.random(k) < 0.9, rng.choice([0.0, -0.0], k), x[r])
        elif what == 3:
            x[r] = rng.integers(-3, 4, k) * 2.0 ** -149
        elif what == 4:
            x[r] = rng.choice([-1.0, 1.0], k) * 3.4e38 * rng.random(k)
        elif what == 5:
            x[r] = rng.normal(0, 1, k) * 2.0 ** -124
        elif what == 6:
            x[r] = rng.normal(0, 1, k) * np.exp(rng.normal(0, 4, k))
    return x


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,k,gap", [(1, 1, 0), (2, 31, 0), (3, 32, 5), (1, 33, 0), (8, 127, 1), (9, 128, 0), (5, 129, 3),
                                     (4, 512, 8), (3, 513, 0), (17, 1000, 24), (8, 4104, 0), (1, 16384, 0)])
def test_quantize(hip, kind, n, k, gap):
    rng = np.random.default_rng(n * 100003 + k)
    with np.errstate(over="ignore"):
        t, x = R.as_type(hard_values(rng, n, k), kind)
    codes, scales = run_quantize(hip, t, kind, k + gap)
    want_codes, want_scales = M.quantize(x)
    assert np.array_equal(scales.cpu().numpy(), want_scales)
    assert np.array_equal(codes.cpu().numpy(), want_codes)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_quantize_not_finite(hip, kind):
    """A block with an infinity or a NaN is NaN; its neighbours are themselves."""
    rng = np.random.default_rng(3)
    x = rng.normal(0, 1, (4, 200))
    x[0, 5], x[1, 32], x[2, 95], x[3, 199] = np.nan, np.inf, -np.inf, np.nan
    t, x = R.as_type(x, kind)
    codes, scales = run_quantize(hip, t, kind, 200)
    want_codes, want_scales = M.quantize(x)
    assert (want_scales == 255).sum() == 4
    assert np.array_equal(scales.cpu().numpy(), want_scales) and np.array_equal(codes.cpu().numpy(), want_codes)


def test_quantize_every_border(hip):
    """Every multiple of 1/16 up to 8, at every exponent a scale can have."""
    v = np.arange(-128, 129) / 16.0
    x = np.zeros((254, 9 * 32))
    for i, e in enumerate(range(-127, 127)):
        part = v * 2.0 ** e
        part = part[np.abs(part) < 3.4e38]
        x[i, :288] = 0
        for b in range(9):
            take = part[31 * b:31 * b + 31]
            x[i, 32 * b:32 * b + len(take)] = take
            x[i, 32 * b + 31] = min(6.0 * 2.0 ** e, 3e38)
    t, x = R.as_type(x, "f32")
    codes, scales = run_quantize(hip, t, "f32", 288)
    want_codes, want_scales = M.quantize(x)
    assert np.array_equal(scales.cpu().numpy(), want_scales) and np.array_equal(codes.cpu().numpy(), want_codes)


def run_dequantize(hip, codes, scales, k, kind, stride):
    n = len(codes)
    out = torch.full((n, stride), 77.0, dtype=R.TORCH[kind], device="cuda")
    c, s = dev(codes), dev(scales)
    hip.dequantize_mxfp4_dev(c.data_ptr(), c.numel(), s.data_ptr(), s.numel(), out.data_ptr(),
                             (n - 1) * stride + k, stride, n, k, R.GGML[kind], stream())
    return out.cpu()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,k,gap", [(256, 32, 0), (3, 1, 2), (5, 131, 0), (7, 1000, 24), (2, 16384, 8), (33, 45, 19)])
def test_dequantize(hip, kind, n, k, gap):
    rng = np.random.default_rng(n + k)
    codes, scales = M.random_rows(rng, n, k, 0, 255)
    if n == 256:
        scales[:, 0] = np.arange(256)
    got = run_dequantize(hip, codes, scales, k, kind, k + gap)
    with np.errstate(over="ignore"):
        exact = torch.from_numpy(M.values(codes, scales, k))
        # what f32 holds, rounded once more
        want = exact.float().to(R.TORCH[kind])
    assert torch.equal(torch.nan_to_num(got[:, :k], nan=12345.0), torch.nan_to_num(want, nan=12345.0))
    assert torch.equal(torch.isnan(got[:, :k]), torch.isnan(want))
    assert (got[:, k:] == 77.0).all()


class Product:
    def __init__(self, hip, t, k, n, kx="f32", ky="f32", bias=False, x_gap=0, y_gap=0, low=118, high=124, seed=0):
        self.rng = rng = np.random.default_rng(seed + t * 7 + k * 13 + n)
        self.hip, self.t, self.k, self.n, self.kx, self.ky = hip, t, k, n, kx, ky
        self.w, self.ws = M.random_rows(rng, n, k, low, high)
        self.bias = rng.normal(0, 1, n).astype(np.float32) if bias else None
        x = rng.normal(0, 1, (t, k)) * (1.0 + 20.0 * (rng.random(k) < 0.01))
        self.xt, self.x = R.as_type(x, kx)
        self.d = {"w": dev(self.w), "ws": dev(self.ws)}
        self.d["x"], self.span = rows(self.xt, k + x_gap)
        self.x_stride, self.y_stride = k + x_gap, n + y_gap
        if bias:
            self.d["bias"] = dev(self.bias)
        self.work = torch.full((max(1, hip.mxfp4_work_bytes(t, k, n)),), 0xCD, dtype=torch.uint8, device="cuda")
        self.out = torch.full((t, self.y_stride), 77.0, dtype=R.TORCH[ky], device="cuda")

    def head(self, out):
        d, n = self.d, self.n
        return (out.data_ptr(), (self.t - 1) * self.y_stride + n, self.y_stride, d["w"].data_ptr(), d["w"].numel(),
                d["ws"].data_ptr(), d["ws"].numel(), d["bias"].data_ptr() if self.bias is not None else 0,
                n if self.bias is not None else 0)

    def oneshot(self):
        self.hip.matmul_mxfp4_dev(*self.head(self.out), self.d["x"].data_ptr(), self.span, self.x_stride,
                                  self.work.data_ptr(), self.work.numel(), self.t, self.k, self.n, R.GGML[self.kx],
                                  R.GGML[self.ky], stream())
        return self.out

    def prequant(self, codes, scales):
        out = torch.full_like(self.out, 77.0)
        self.hip.matmul_mxfp4_prequant_dev(*self.head(out), codes.data_ptr(), codes.numel(), scales.data_ptr(),
                                           scales.numel(), self.work.data_ptr(), self.work.numel(), self.t, self.k,
                                           self.n, R.GGML[self.ky], stream())
        return out

    def check(self, out, codes, scales):
        """Steps of 128 products are exact sums rounded to f32 with what was there, off by
        at most 2^-23 of the terms' magnitudes; joins of up to 16 parts and the bias as
        much each; then the output's rounding."""
        bias = None if self.bias is None else self.bias.astype(np.float64)
        want, size = M.product(M.values(codes, scales, self.k), M.values(self.w, self.ws, self.k), bias)
        tol = ((self.k + 127) // 128 + 17) * 2.0 ** -23 * size + M.rounding(want, self.ky)
        got = out[:, :self.n].cpu().double().numpy()
        assert np.array_equal(np.isnan(got), np.isnan(want))
        bad = ~(np.abs(got - want) <= tol) & ~np.isnan(want)
        assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], tol[bad][:5])
        assert (out[:, self.n:] == 77.0).all()

    def both(self):
        """The two forms give the same, and what they should."""
        codes, scales = M.quantize(self.x)
        out = self.oneshot()
        assert torch.equal(torch.nan_to_num(out), torch.nan_to_num(self.prequant(dev(codes), dev(scales))))
        self.check(out, codes, scales)


SIZES = [(1, 1, 1), (1, 32, 16), (2, 33, 17), (1, 100, 40), (3, 127, 15), (4, 128, 64), (5, 129, 65), (7, 600, 130),
         (8, 512, 96), (13, 1000, 33), (16, 2048, 48), (17, 513, 200), (31, 300, 31), (32, 1024, 128), (33, 640, 257),
         (48, 256, 72), (64, 768, 64), (77, 2000, 101), (100, 1025, 300), (128, 512, 128), (129, 384, 129),
         (200, 896, 520), (256, 1152, 256), (300, 160, 1000), (1, 4096, 1000), (1, 14000, 48), (2, 7168, 130)]


@pytest.mark.parametrize("t,k,n", SIZES)
def test_product(hip, t, k, n):
    kinds = ["f32", "f16", "bf16"]
    i = t + k + n
    Product(hip, t, k, n, kinds[i % 3], kinds[i // 3 % 3], bias=i % 2 == 0, x_gap=[0, 3, 64][i % 3],
            y_gap=[0, 8, 5][i // 2 % 3]).both()


@pytest.mark.parametrize("t", [1, 5, 40, 150])
@pytest.mark.parametrize("low,high", [(100, 160), (0, 3), (126, 254)])
def test_product_of_wide_scales(hip, t, low, high):
    """Scales over the whole range: sums that lose what is small beside them, and ones
    that f32 cannot hold."""
    p = Product(hip, t, 700, 90, low=low, high=high)
    codes, scales = M.random_rows(np.random.default_rng(t), t, 700, 100, 130)
    M.clear_tail(codes, 700)
    out = p.prequant(dev(codes), dev(scales))
    want, size = M.product(M.values(codes, scales, 700), M.values(p.w, p.ws, 700), None)
    got = out.cpu().double().numpy()
    fits = size < 3e38
    tol = (6 + 17) * 2.0 ** -23 * size + M.rounding(want, "f32") + 700 * 2.0 ** -126
    assert (np.abs(got - want)[fits] <= tol[fits]).all()
    assert fits.any()


@pytest.mark.parametrize("t", [1, 3, 20, 80, 200])
def test_product_not_finite(hip, t):
    """A NaN block is NaN in its own token's or channel's outputs and no other's."""
    p = Product(hip, t, 300, 50)
    p.ws[7, 2] = 255
    p.d["ws"] = dev(p.ws)
    p.x[t // 2, 290] = np.inf
    p.xt = torch.from_numpy(p.x.astype(np.float32))
    p.d["x"], p.span = rows(p.xt, 300)
    p.both()


@pytest.mark.parametrize("t", [1, 4, 33, 130])
def test_product_on_another_stream_and_in_a_graph(hip, t):
    p = Product(hip, t, 1100, 200, "bf16", "bf16", bias=True)
    want = p.oneshot().clone()
    codes, scales = M.quantize(p.x)
    p.check(want, codes, scales)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        p.out.fill_(77.0)
        p.oneshot()
    side.synchronize()
    assert torch.equal(p.out, want)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        p.oneshot()
    for i in range(4):
        p.d["x"].mul_(-1.0 if i % 2 == 0 else -2.0)  # (powers of two: the codes are the same)
        p.out.fill_(77.0)
        p.work.fill_(i)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        again = p.out.clone()
        p.out.fill_(77.0)
        assert torch.equal(again, p.oneshot())


@pytest.mark.parametrize("t", [1, 40])
def test_product_beyond_32_bit_offsets(hip, t):
    """Weights of more than 2^32 bytes: rows at the end as those at the start."""
    k, n = 65536, 133000
    assert n * M.row_bytes(k) > 1 << 32
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    few = torch.randint(0, 256, (1000, M.row_bytes(k)), dtype=torch.uint8, device="cuda", generator=g)
    fs = torch.randint(110, 116, (1000, M.scale_bytes(k)), dtype=torch.uint8, device="cuda", generator=g)
    w, ws = few.repeat(133, 1), fs.repeat(133, 1)
    x = torch.randn(t, k, device="cuda", generator=g)
    out = torch.full((t, n), 77.0, device="cuda")
    small = torch.full((t, 1000), 77.0, device="cuda")
    for o, a, b, m in ((out, w, ws, n), (small, few, fs, 1000)):
        work = torch.empty(hip.mxfp4_work_bytes(t, k, m), dtype=torch.uint8, device="cuda")
        hip.matmul_mxfp4_dev(o.data_ptr(), o.numel(), m, a.data_ptr(), a.numel(), b.data_ptr(), b.numel(), 0, 0,
                             x.data_ptr(), x.numel(), k, work.data_ptr(), work.numel(), t, k, m, 0, 0, stream())
    codes, scales = run_quantize(hip, x.cpu(), "f32", k)
    v = M.values(codes.cpu().numpy(), scales.cpu().numpy(), k)
    want, size = M.product(v, M.values(few[:64].cpu().numpy(), fs[:64].cpu().numpy(), k), None)
    tol = torch.from_numpy((512 + 17) * 2.0 ** -23 * size + M.rounding(want, "f32"))
    got = out.view(t, 133, 1000)[:, :, :64].cpu().double()
    assert (torch.abs(got - torch.from_numpy(want)[:, None, :]) <= tol[:, None, :]).all()
    assert (torch.abs(small[:, :64].cpu().double() - torch.from_numpy(want)) <= tol).all()
