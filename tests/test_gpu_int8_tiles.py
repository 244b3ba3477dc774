"""Every kernel of the int8 product against whole-number arithmetic, bit for bit.

Scales are powers of two and sums below 2^24, so every f32 step before the bias is
exact; the bias and the output's type round once each, as they do in the
reference. test_int8_launch.py shows that each size runs the kernel it stands for."""
import pytest
import torch

import serving_ref as R
from int8_cases import CASES

pytestmark = pytest.mark.gpu

#: x's type, the output's type, a bias, how far apart rows lie beyond their length
#: (x, out), elements before the first (wscale, bias, out)
FORMS = [("f32", "f32", False, (0, 0), 0), ("bf16", "bf16", True, (3, 1), 0), ("f16", "f16", True, (0, 4), 1),
         ("f32", "bf16", False, (8, 64), 0), ("bf16", "f32", True, (1, 3), 1)]


@pytest.mark.parametrize("tile,n_tok,n,out_dim", CASES, ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else None)
def test_bit_for_bit(hip, tile, n_tok, n, out_dim):
    g = torch.Generator(device="cuda").manual_seed(n_tok * 131 + n)

    def ints(lo, hi, *shape):
        return torch.randint(lo, hi + 1, shape, device="cuda", generator=g)
    row, most = hip.int8_row_bytes(n), min(127, (1 << 24) // (127 * n) - 1)
    codes = ints(-127, 127, n_tok, n)
    codes[torch.arange(n_tok, device="cuda"), ints(0, n - 1, n_tok)] = 127  # so the scale is what follows
    xscale = torch.exp2(ints(-3, 3, n_tok).float())
    w = torch.full((out_dim, row), 77, dtype=torch.int8, device="cuda")  # (what lies behind a row does not matter)
    w[:, :n] = ints(-most - 1 if most == 127 else -most, most, out_dim, n).to(torch.int8)
    ws = torch.exp2(ints(-12, -9, out_dim).float())
    bias = torch.round(torch.randn(out_dim, device="cuda", generator=g) * 2.0 ** 20) * 2.0 ** -20
    sums = torch.matmul(codes.double(), w[:, :n].double().t().contiguous())
    assert sums.abs().max() < 1 << 24
    product = (sums * xscale[:, None].double() * ws[None, :].double()).float()
    del sums
    st = torch.cuda.current_stream().cuda_stream
    for dtype_x, dtype_out, has_bias, (xpad, opad), before in FORMS:
        # (both below 2^19 and multiples of 2^-20: their sum is exact in 64 bits)
        want = (product.double() + bias.double()[None, :]).float() if has_bias else product
        want = want.to(R.TORCH[dtype_out])
        x = torch.full((n_tok, n + xpad), float("nan"), dtype=R.TORCH[dtype_x], device="cuda")
        x[:, :n] = (codes.float() * xscale[:, None]).to(x.dtype)  # (at most 8 bits: exact)
        stride = out_dim + opad
        out = torch.full((2, before + n_tok * stride + 8), -7.0, dtype=R.TORCH[dtype_out], device="cuda")
        at = torch.cat([torch.zeros(before, device="cuda"), ws]), torch.cat([torch.zeros(before, device="cuda"), bias])
        work = torch.empty(hip.int8_work_bytes(n_tok, n, out_dim), dtype=torch.uint8, device="cuda")
        xq, sc = torch.full((n_tok, row), 99, dtype=torch.int8, device="cuda"), torch.zeros(n_tok, device="cuda")
        wsp, bp, bl = at[0].data_ptr() + 4 * before, at[1].data_ptr() + 4 * before, out_dim
        if not has_bias:
            bp = bl = 0
        out_len = (n_tok - 1) * stride + out_dim
        x_len = (n_tok - 1) * (n + xpad) + n
        op = [o.data_ptr() + before * o.element_size() for o in out]
        hip.quantize_int8_dev(x.data_ptr(), x_len, n + xpad, xq.data_ptr(), xq.numel(), sc.data_ptr(), n_tok,
                              n_tok, n, R.GGML[dtype_x], st)
        hip.matmul_int8_prequant_dev(op[0], out_len, stride, w.data_ptr(), w.numel(), wsp, out_dim, bp, bl,
                                     xq.data_ptr(), xq.numel(), sc.data_ptr(), n_tok, 0, 0, n_tok, n, out_dim,
                                     R.GGML[dtype_out], st)
        hip.matmul_int8_dev(op[1], out_len, stride, w.data_ptr(), w.numel(), wsp, out_dim, bp, bl, x.data_ptr(),
                            x_len, n + xpad, work.data_ptr(), work.numel(), n_tok, n, out_dim, R.GGML[dtype_x],
                            R.GGML[dtype_out], st)
        torch.cuda.synchronize()
        assert torch.equal(sc, xscale)
        assert torch.equal(xq[:, :n].int(), codes.int()) and not xq[:, n:].any()
        for o in out:
            assert (o[:before] == -7.0).all() and (o[before + n_tok * stride:] == -7.0).all()
            o = o[before:before + n_tok * stride].view(n_tok, stride)
            assert (o[:, out_dim:] == -7.0).all(), "wrote between the rows"
            bad = (o[:, :out_dim] != want).nonzero()
            assert not len(bad), (dtype_x, dtype_out, len(bad), bad[:4].tolist(), bad[-4:].tolist())
