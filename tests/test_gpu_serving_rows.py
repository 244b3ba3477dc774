"""As many rows as a call of routing, the int8 quantiser and the log-probabilities
takes: every row, against torch in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

ROWS = (1 << 23) - 1


def stream():
    return torch.cuda.current_stream().cuda_stream


def test_route(hip):
    x = torch.randint(-40, 40, (ROWS, 2), device="cuda").float() / 8
    ids = torch.full((ROWS, 1), -5, dtype=torch.int32, device="cuda")
    w = torch.zeros(ROWS, 1, device="cuda")
    hip.moe_route_dev(ids.data_ptr(), w.data_ptr(), ROWS, x.data_ptr(), 2 * ROWS, 2, 0, 0, ROWS, 2, 1, 1, 1, 1,
                      1, False, 1.0, 0, stream())
    assert torch.equal(ids[:, 0], (x[:, 1] > x[:, 0]).int())  # equal ones: the lower id
    want = torch.sigmoid(x.double()).amax(1)
    # one rounding to f32, half a step, and what 64-bit sums leave beside it
    assert ((w[:, 0].double() - want).abs() <= want * (2.0**-24 + 2.0**-48)).all()


def test_quantize(hip):
    x = torch.randint(-127, 128, (ROWS, 2), device="cuda").float()
    x[:, 0] = 127.0  # the scale is 1, the codes are the values
    codes = torch.full((ROWS, 64), 99, dtype=torch.int8, device="cuda")
    scale = torch.zeros(ROWS, device="cuda")
    hip.quantize_int8_dev(x.data_ptr(), 2 * ROWS, 2, codes.data_ptr(), codes.numel(), scale.data_ptr(), ROWS, ROWS, 2,
                          0, stream())
    assert (scale == 1.0).all()
    assert torch.equal(codes[:, :2].float(), x)
    assert not codes[:, 2:].any()


def test_logprobs(hip):
    x = torch.randn(ROWS, 2, device="cuda")
    tok = torch.randint(0, 2, (ROWS,), dtype=torch.int32, device="cuda")
    lp, rank = torch.zeros(ROWS, device="cuda"), torch.zeros(ROWS, dtype=torch.int32, device="cuda")
    assert hip.token_logprobs_work_bytes(ROWS, 2, 0) == 0
    hip.token_logprobs_dev(lp.data_ptr(), 0, rank.data_ptr(), ROWS, 0, 0, 0, x.data_ptr(), 2 * ROWS, 2, tok.data_ptr(),
                           ROWS, 0, 0, ROWS, 2, 0, 0, stream())
    mine, other = x.gather(1, tok[:, None].long())[:, 0], x.gather(1, 1 - tok[:, None].long())[:, 0]
    assert torch.equal(rank, 1 + (other > mine).int())
    want = torch.log_softmax(x.double(), 1).gather(1, tok[:, None].long())[:, 0]
    # l - m is rounded once (half a step of it); S = 1 + e in (1, 2], e by an exp of
    # few steps' error and the sum rounded, so log S is off by at most 4 steps of 1 and
    # its own rounding; the difference is rounded once more
    tol = 2.0**-24 * (2 * want.abs() + (x[:, 0] - x[:, 1]).abs().double() + 8)
    assert ((lp.double() - want).abs() <= tol).all()
