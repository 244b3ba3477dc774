"""Replays of the 4-bit mixture-of-experts layer with rows that are NaN: such a row has to be
written as NaN each time, too, and the others have the eager run's bits."""
import numpy as np
import pytest
import torch

from moe_layer_cases import PART_CASES
from test_gpu_moe_layer import CASES, Layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", PART_CASES + [c for c in CASES if 2 < c["t"] < 17][:4],
                         ids=lambda c: "-".join(str(c.get(n)) for n in ("t", "embd", "ff", "experts", "k")))
def test_rows_of_nan_are_written_by_every_replay(hip, case):
    p = Layer(hip, **case)
    last = case["t"] - 1
    p.x[0, -1], p.x[last, 0] = np.inf, np.nan
    p.xt = torch.from_numpy(p.x).to(p.xt.dtype)
    p.upload()
    p.run()
    # (not p.check(): weights of a token with an infinity can be inf / inf)
    ids, weights, out, tol = p.want()
    got_w, got = p.weights.cpu().double().numpy(), p.out[:, :case["embd"]].cpu().double().numpy()
    assert np.array_equal(p.ids.cpu().numpy(), ids)
    for a, b, off in ((got_w, weights, np.abs(weights) * (2.0 ** -24 + 2.0 ** -45) + 2.0 ** -150), (got, out, tol)):
        assert np.array_equal(np.isnan(a), np.isnan(b))
        with np.errstate(invalid="ignore"):
            assert ((np.abs(a - b) <= off) | (a == b) | np.isnan(b)).all()
    want = p.out.clone()
    assert torch.isnan(want[[0, last], :case["embd"]]).all()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        p.run()
    for fill in (0.0, 77.0, -1.0):
        p.out.fill_(fill)
        p.out[:, case["embd"]:] = 77.0
        p.work.random_(0, 256)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(torch.isnan(p.out), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(p.out), torch.nan_to_num(want))
