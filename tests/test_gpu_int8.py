"""rsllm_hip_quantize_int8_dev, _matmul_int8_prequant_dev and _matmul_int8_dev
against 64-bit arithmetic: codes and scales equal, products within the roundings
of the formula (three to f32, one more with a bias, one to the output's type)."""
import numpy as np
import pytest
import torch

import serving_ref as R

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")
KINDS = ["f32", "f16", "bf16"]


def quantize(hip, x, dtype="f32", stride=None):
    """(the codes with their padding, scales, the values in 64 bits)."""
    t, values = R.as_type(x, dtype)
    n_tok, n = t.shape
    buf, span = R.strided(t, stride or n)
    d, row = buf.cuda(), hip.int8_row_bytes(n)
    xq = torch.full((n_tok * row + 64,), 77, dtype=torch.int8, device="cuda")
    sc = torch.full((n_tok + 4,), -7.0, device="cuda")
    hip.quantize_int8_dev(d.data_ptr(), span, stride or n, xq.data_ptr(), n_tok * row, sc.data_ptr(),
                          n_tok, n_tok, n, R.GGML[dtype], torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert (xq[n_tok * row:] == 77).all() and (sc[n_tok:] == -7.0).all()
    return xq[:n_tok * row].view(n_tok, row), sc[:n_tok], values


def check_codes(hip, x, dtype="f32", stride=None):
    xq, sc, values = quantize(hip, x, dtype, stride)
    codes, scales = R.quantize(values)
    n = values.shape[1]
    np.testing.assert_array_equal(sc.cpu().numpy(), scales)
    np.testing.assert_array_equal(xq[:, :n].cpu().numpy(), codes)
    assert (xq[:, n:] == 0).all()


@pytest.mark.parametrize("dtype", KINDS)
@pytest.mark.parametrize("n_tok,n,stride", [
    (1, 1, None), (3, 63, None), (2, 64, 67), (5, 100, None), (1, 4096, None), (33, 1000, 1001),
    (7, 8192, 8200), (2, 14336, None), (1, 40001, None), (1, 131071, None), (300, 257, 264)])
def test_quantise_sizes(hip, dtype, n_tok, n, stride):
    rng = np.random.default_rng(n_tok * n)
    x = rng.normal(0, 1, (n_tok, n)) * np.exp(rng.normal(0, 2, (n_tok, 1)))
    check_codes(hip, x, dtype, stride)


def test_quantise_halves_and_their_neighbours(hip):
    """Quotients of exactly k + 1/2 (to even) and one f32 step to either side."""
    for d in (1.0, 0.75, 3.1415927, 1e-30, 2e30):
        d = np.float32(np.float32(d * 127) / np.float32(127))
        x = [np.float32(127 * np.float64(d))]
        for k in range(-126, 126):
            h = np.float32((k + 0.5) * np.float64(d))
            x += [h, np.nextafter(h, np.float32(INF)), np.nextafter(h, np.float32(-INF))]
        check_codes(hip, np.array([x]), "f32")


def test_quantise_extremes(hip):
    big, tiny = np.float32(3.4e38), np.float32(2.0 ** -149)
    rows = [np.zeros(70), np.full(70, big), np.full(70, -big), np.r_[big, np.full(69, 1e-38)],
            np.full(70, tiny), np.r_[np.arange(1, 71) * tiny], np.r_[np.arange(70) * 3 * tiny],
            np.r_[64 * tiny, np.full(69, 32 * tiny)], np.r_[np.arange(70) * 200 * tiny],
            np.linspace(-1e-37, 1e-37, 70), np.full(70, -0.0)]
    check_codes(hip, np.array(rows, np.float32), "f32")
    check_codes(hip, np.array([[65504.0, -65504.0, 6e-8, 0.0], [6e-8, -6e-8, 1.2e-7, 3e-5]]), "f16")
    check_codes(hip, np.array([[3.3e38, 1.0, 2.0, -5e37]]), "bf16")


def test_quantise_non_finite_rows_are_nan_and_alone(hip):
    rng = np.random.default_rng(3)
    x = rng.normal(0, 1, (6, 500))
    x[1, 499], x[3, 0], x[4, 77] = NAN, INF, -INF
    for dtype in KINDS:
        xq, sc, values = quantize(hip, x, dtype)
        codes, scales = R.quantize(values)
        np.testing.assert_array_equal(sc.cpu().numpy(), scales)
        np.testing.assert_array_equal(xq[:, :500].cpu().numpy(), codes)
        assert np.isnan(scales[[1, 3, 4]]).all() and (codes[[1, 3, 4]] == 0).all()


def weights(rng, out_dim, in_dim, fill=0):
    row = (in_dim + 63) // 64 * 64
    w = rng.integers(-127, 128, (out_dim, row)).astype(np.int8)
    w[:, in_dim:] = fill
    return w, (rng.random(out_dim).astype(np.float32) + np.float32(0.5)) / np.float32(73 * in_dim ** 0.5)


def product(hip, x, w, ws, bias=None, dtype_x="f32", dtype_out="f32", x_stride=None, out_stride=None,
            stream=None):
    """Both forms on the same inputs: their outputs bit for bit alike, and within
    the roundings of the 64-bit result."""
    t, values = R.as_type(x, dtype_x)
    n_tok, n = t.shape
    out_dim, row = w.shape
    xb, span = R.strided(t, x_stride or n)
    xd, wd, wsd = xb.cuda(), torch.from_numpy(w).cuda(), torch.from_numpy(ws).cuda()
    bd = None if bias is None else torch.from_numpy(bias).cuda()
    os_ = out_stride or out_dim
    work = torch.full((hip.int8_work_bytes(n_tok, n, out_dim),), 0xAB, dtype=torch.uint8, device="cuda")
    mark = -7.0
    outs = [torch.full((n_tok * os_ + 16,), mark, dtype=R.TORCH[dtype_out], device="cuda") for _ in range(2)]
    out_len = (n_tok - 1) * os_ + out_dim
    st = stream or torch.cuda.current_stream().cuda_stream
    bp, bl = (0, 0) if bd is None else (bd.data_ptr(), out_dim)
    torch.cuda.synchronize()
    hip.matmul_int8_dev(outs[0].data_ptr(), out_len, os_, wd.data_ptr(), wd.numel(), wsd.data_ptr(),
                        out_dim, bp, bl, xd.data_ptr(), span, x_stride or n, work.data_ptr(),
                        work.numel(), n_tok, n, out_dim, R.GGML[dtype_x], R.GGML[dtype_out], st)
    xq = torch.empty(n_tok, row, dtype=torch.int8, device="cuda")
    sc = torch.empty(n_tok, device="cuda")
    hip.quantize_int8_dev(xd.data_ptr(), span, x_stride or n, xq.data_ptr(), xq.numel(), sc.data_ptr(),
                          n_tok, n_tok, n, R.GGML[dtype_x], st)
    hip.matmul_int8_prequant_dev(outs[1].data_ptr(), out_len, os_, wd.data_ptr(), wd.numel(),
                                 wsd.data_ptr(), out_dim, bp, bl, xq.data_ptr(), xq.numel(),
                                 sc.data_ptr(), n_tok, work.data_ptr(), work.numel(), n_tok, n,
                                 out_dim, R.GGML[dtype_out], st)
    torch.cuda.synchronize()
    codes, scales = R.quantize(values)
    want, p = R.int8_product(codes, scales, w[:, :n], ws, bias)
    raw = [o.cpu() for o in outs]
    assert torch.equal(raw[0].view(torch.uint8), raw[1].view(torch.uint8)), "the two forms differ"
    got = raw[0][:n_tok * os_].view(n_tok, os_).double().numpy()
    assert (got[:, out_dim:] == mark).all(), "wrote between the rows"
    assert (raw[0][n_tok * os_:].double().numpy() == mark).all(), "wrote behind the last row"
    got = got[:, :out_dim]
    with np.errstate(invalid="ignore"):
        assert np.array_equal(np.isnan(got), np.isnan(want))
        # f32(acc), * d, * wscale; + bias; the output's type
        bound = 3.001 * 2.0 ** -24 * np.abs(p) + 2.0 ** -24 * np.abs(want) * (bias is not None) \
            + 1.001 * R.HALF_STEP[dtype_out] * np.abs(want) * (dtype_out != "f32") + R.TINY_STEP[dtype_out]
        assert not (np.abs(got - want) > bound).any(), np.nanmax(np.abs(got - want) / bound)
    return got


@pytest.mark.parametrize("n_tok", [1, 2, 3, 4, 5, 8, 9, 15, 16, 17, 31, 32, 33, 48, 64, 65, 100, 127,
                                   128, 129, 200, 255, 256, 257, 300, 511, 700])
@pytest.mark.parametrize("in_dim,out_dim", [(64, 16), (100, 40), (256, 129), (1000, 333), (448, 640)])
def test_token_counts(hip, n_tok, in_dim, out_dim):
    rng = np.random.default_rng(n_tok * 1000 + out_dim)
    w, ws = weights(rng, out_dim, in_dim, fill=55)
    product(hip, rng.normal(0, 1, (n_tok, in_dim)), w, ws)


@pytest.mark.parametrize("n_tok,in_dim,out_dim", [
    (1, 1, 1), (1, 131071, 3), (2, 63, 7), (4, 14336, 513), (6, 8200, 1000), (20, 4097, 100),
    (1, 4096, 4096), (1, 2048, 16384), (7, 4096, 1024), (16, 14336, 512), (32, 4096, 1024),
    (40, 128, 20000), (96, 2048, 1000), (130, 4096, 260), (520, 640, 1100), (1030, 576, 300),
    (2048, 192, 128), (3, 192, 40000), (256, 16384, 256)])
def test_shapes(hip, n_tok, in_dim, out_dim):
    rng = np.random.default_rng(in_dim + out_dim)
    w, ws = weights(rng, out_dim, in_dim, fill=-3)
    product(hip, rng.normal(0, 1, (n_tok, in_dim)), w, ws,
            bias=rng.normal(0, 1, out_dim).astype(np.float32))


@pytest.mark.parametrize("dtype_out", KINDS)
@pytest.mark.parametrize("dtype_x", KINDS)
@pytest.mark.parametrize("n_tok", [1, 3, 12, 50, 260])
def test_types(hip, n_tok, dtype_x, dtype_out):
    rng = np.random.default_rng(n_tok)
    w, ws = weights(rng, 200, 320)
    product(hip, rng.normal(0, 1, (n_tok, 320)), w, ws, dtype_x=dtype_x, dtype_out=dtype_out,
            bias=rng.normal(0, 1, 200).astype(np.float32))


@pytest.mark.parametrize("dtype_out", ["f32", "bf16"])
@pytest.mark.parametrize("n_tok", [1, 4, 19, 70, 300])
def test_strided_rows(hip, n_tok, dtype_out):
    rng = np.random.default_rng(n_tok)
    w, ws = weights(rng, 130, 200)
    for xs, os_ in ((201, 131), (264, 192), (200, 1001)):
        product(hip, rng.normal(0, 1, (n_tok, 200)), w, ws, x_stride=xs, out_stride=os_,
                dtype_out=dtype_out)


@pytest.mark.parametrize("n_tok", [1, 4, 13, 64, 200, 300])
def test_largest_sums(hip, n_tok):
    """Codes of -128 and +-127 throughout: the sums come within one code of the
    32-bit border at the longest rows."""
    n = 131071 if n_tok <= 64 else 4096
    w = np.full((18, (n + 63) // 64 * 64), -128, np.int8)
    w[1::3], w[2::3, ::2] = 127, 127
    x = np.ones((n_tok, n))
    x[::2] = -1.0
    product(hip, x, w, np.full(18, 1e-3, np.float32))


@pytest.mark.parametrize("n_tok", [2, 4, 20, 100, 300])
def test_non_finite_tokens_stay_alone(hip, n_tok):
    rng = np.random.default_rng(n_tok)
    w, ws = weights(rng, 96, 192)
    x = rng.normal(0, 1, (n_tok, 192))
    x[0, 5], x[n_tok - 1, 191] = NAN, INF
    got = product(hip, x, w, ws)
    assert np.isnan(got[[0, n_tok - 1]]).all()
    x[:] = 0.0
    got = product(hip, x, w, ws)
    assert (got == 0).all()


@pytest.mark.parametrize("n_tok", [1, 4, 20, 70, 300])
@pytest.mark.parametrize("dtype_out", KINDS)
def test_scales_and_outputs_aligned_to_their_elements_alone(hip, n_tok, dtype_out):
    """wscale, bias and out one element into an allocation, so on no 16-byte
    border; work of the halves' product left out."""
    rng = np.random.default_rng(n_tok)
    n, out_dim = 192, 132
    w, ws = weights(rng, out_dim, n)
    bias = rng.normal(0, 1, out_dim).astype(np.float32)
    codes, scales = R.quantize(rng.normal(0, 1, (n_tok, n)).astype(np.float32).astype(np.float64))
    want, p = R.int8_product(codes, scales, w[:, :n], ws, bias)

    def shifted(a):
        return torch.cat([torch.full((1,), 9.0), torch.from_numpy(a)]).cuda()
    wd, xq, sc = torch.from_numpy(w).cuda(), torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda()
    wsd, bd = shifted(ws), shifted(bias)
    y = torch.full((1 + n_tok * out_dim,), -7.0, dtype=R.TORCH[dtype_out], device="cuda")
    hip.matmul_int8_prequant_dev(y.data_ptr() + y.element_size(), n_tok * out_dim, out_dim, wd.data_ptr(),
                                 wd.numel(), wsd.data_ptr() + 4, out_dim, bd.data_ptr() + 4, out_dim,
                                 xq.data_ptr(), xq.numel(), sc.data_ptr(), n_tok, 0, 0, n_tok, n, out_dim,
                                 R.GGML[dtype_out], torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    got = y.cpu().double().numpy()
    assert got[0] == -7.0
    got = got[1:].reshape(n_tok, out_dim)
    bound = 3.001 * 2.0 ** -24 * np.abs(p) + 2.0 ** -24 * np.abs(want) \
        + 1.001 * R.HALF_STEP[dtype_out] * np.abs(want) * (dtype_out != "f32") + R.TINY_STEP[dtype_out]
    assert not (np.abs(got - want) > bound).any()


@pytest.mark.parametrize("n_tok", [1, 3, 20, 70])
def test_weights_beyond_32_bit_offsets(hip, n_tok):
    """A matrix of 5.2 GB: the last rows against their own products."""
    n, out_dim, tail = 131071, 40000, 50
    w = torch.randint(-127, 128, (out_dim, 131072), dtype=torch.int8, device="cuda")
    ws = torch.full((out_dim,), 1e-6, device="cuda")
    x = torch.randn(n_tok, n, device="cuda")
    y = torch.full((n_tok, out_dim), NAN, device="cuda")
    work = torch.empty(hip.int8_work_bytes(n_tok, n, out_dim), dtype=torch.uint8, device="cuda")
    hip.matmul_int8_dev(y.data_ptr(), y.numel(), out_dim, w.data_ptr(), w.numel(), ws.data_ptr(), out_dim,
                        0, 0, x.data_ptr(), x.numel(), n, work.data_ptr(), work.numel(), n_tok, n, out_dim,
                        stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    codes, scales = R.quantize(x.cpu().double().numpy())
    want, p = R.int8_product(codes, scales, w[-tail:, :n].cpu().numpy(), ws[-tail:].cpu().numpy(), None)
    got = y.cpu().double().numpy()
    assert np.isfinite(got).all()
    assert not (np.abs(got[:, -tail:] - want) > 3.001 * 2.0 ** -24 * np.abs(p)).any()


def test_overflow_to_the_output_type(hip):
    """A product above f16's largest is inf, as a rounding gives."""
    w = np.full((4, 64), 127, np.int8)
    x = np.full((3, 64), 1e4)
    t = torch.from_numpy(x.astype(np.float32)).cuda()
    y = torch.zeros(3, 4, dtype=torch.float16, device="cuda")
    wd, ws = torch.from_numpy(w).cuda(), torch.ones(4, device="cuda")
    work = torch.empty(hip.int8_work_bytes(3, 64, 4), dtype=torch.uint8, device="cuda")
    hip.matmul_int8_dev(y.data_ptr(), 12, 4, wd.data_ptr(), 256, ws.data_ptr(), 4, 0, 0, t.data_ptr(),
                        192, 64, work.data_ptr(), work.numel(), 3, 64, 4, 0, 1)
    torch.cuda.synchronize()
    assert torch.isinf(y).all()


@pytest.mark.parametrize("n_tok", [1, 8, 200])
def test_a_token_is_the_same_in_any_batch(hip, n_tok):
    """The sums are whole numbers, so a token's outputs do not depend on what it
    is computed with."""
    rng = np.random.default_rng(4)
    w, ws = weights(rng, 300, 2048)
    x = rng.normal(0, 1, (300, 2048))
    every = product(hip, x, w, ws)
    np.testing.assert_array_equal(product(hip, x[:n_tok], w, ws), every[:n_tok])


@pytest.mark.parametrize("n_tok", [1, 6, 40, 300])
def test_on_other_streams_and_captured(hip, n_tok):
    rng = np.random.default_rng(5)
    n, out_dim = 1024, 520
    w, ws = weights(rng, out_dim, n)
    side = torch.cuda.Stream()
    product(hip, rng.normal(0, 1, (n_tok, n)), w, ws, stream=side.cuda_stream)
    wd, wsd = torch.from_numpy(w).cuda(), torch.from_numpy(ws).cuda()
    graphs = []
    before = hip.device_allocations()
    for _ in range(2):  # two graphs, a workspace each, replayed side by side
        x = torch.zeros(n_tok, n, device="cuda")
        y = torch.zeros(n_tok, out_dim, device="cuda")
        work = torch.empty(hip.int8_work_bytes(n_tok, n, out_dim), dtype=torch.uint8, device="cuda")
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            hip.matmul_int8_dev(y.data_ptr(), y.numel(), out_dim, wd.data_ptr(), wd.numel(),
                                wsd.data_ptr(), out_dim, 0, 0, x.data_ptr(), x.numel(), n,
                                work.data_ptr(), work.numel(), n_tok, n, out_dim,
                                stream=torch.cuda.current_stream().cuda_stream)
        graphs.append((x, y, work, g, torch.cuda.Stream()))
    assert hip.device_allocations() == before
    for i in range(4):
        want = []
        for x, y, *_ in graphs:
            v = rng.normal(0, 1, (n_tok, n)).astype(np.float32)
            x.copy_(torch.from_numpy(v))
            y.fill_(NAN)
            codes, scales = R.quantize(v.astype(np.float64))
            want.append(R.int8_product(codes, scales, w, ws, None)[0])
        torch.cuda.synchronize()
        for _, _, _, g, s in graphs:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for (_, y, *_), p in zip(graphs, want):
            got = y.cpu().double().numpy()
            assert not (np.abs(got - p) > 3.001 * 2.0 ** -24 * np.abs(p) + 2.0 ** -150).any()
