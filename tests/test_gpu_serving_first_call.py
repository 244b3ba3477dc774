"""The first call of a process into each kernel of routing, the int8 product and the
log-probabilities may be one that a graph records: nothing is set up by an earlier
eager call. In a process of its own, since this one has called them already."""
import os
import subprocess
import sys

import pytest

CHILD = """
import torch
from rsllm_amd import backend as B
B.init(0)
g = torch.Generator(device="cuda").manual_seed(5)
def rnd(*s): return torch.randn(*s, device="cuda", generator=g)
stream = lambda: torch.cuda.current_stream().cuda_stream
calls = []
def route(t, e, k):
    x, ids, w = rnd(t, e), torch.empty(t, k, dtype=torch.int32, device="cuda"), torch.empty(t, k, device="cuda")
    calls.append((f"route {t} x {e}", [ids, w], lambda: B.moe_route_dev(
        ids.data_ptr(), w.data_ptr(), t * k, x.data_ptr(), t * e, e, 0, 0, t, e, k, 1, 1, 1, 1, True, 1.0, 0, stream())))
def int8(t, k, n):
    rb = B.int8_row_bytes(k)
    x, y, ws = rnd(t, k), torch.empty(t, n, device="cuda"), torch.rand(n, device="cuda", generator=g)
    w = torch.randint(-127, 128, (n, rb), dtype=torch.int8, device="cuda", generator=g)
    work = torch.empty(B.int8_work_bytes(t, k, n), dtype=torch.uint8, device="cuda")
    calls.append((f"int8 {t} x {k} x {n}", [y], lambda: B.matmul_int8_dev(
        y.data_ptr(), t * n, n, w.data_ptr(), n * rb, ws.data_ptr(), n, 0, 0, x.data_ptr(), t * k, k,
        work.data_ptr(), work.numel(), t, k, n, 0, 0, stream())))
def logprobs(t, v, n):
    x, tok = rnd(t, v), torch.zeros(t, dtype=torch.int32, device="cuda")
    lp, en, rk = torch.empty(t, device="cuda"), torch.empty(t, device="cuda"), torch.empty(t, dtype=torch.int32, device="cuda")
    ids, top = torch.empty(t, n, dtype=torch.int32, device="cuda"), torch.empty(t, n, device="cuda")
    work = torch.empty(B.token_logprobs_work_bytes(t, v, n) + 256, dtype=torch.uint8, device="cuda")
    calls.append((f"logprobs {t} x {v}", [lp, en, rk, ids, top], lambda: B.token_logprobs_dev(
        lp.data_ptr(), en.data_ptr(), rk.data_ptr(), t, ids.data_ptr(), top.data_ptr(), t * n, x.data_ptr(),
        t * v, v, tok.data_ptr(), t, work.data_ptr(), work.numel(), t, v, n, 0, stream())))
for t, e in ((3, 64), (3, 128), (3, 256), (3, 512), (3, 1024), (3, 1500)):
    route(t, e, 6)
# one token, few, then the tiles up to the widest
for t, k, n in ((1, 512, 96), (3, 512, 96), (20, 512, 512), (40, 512, 2048), (64, 4096, 4096), (128, 1024, 4096),
                (300, 1024, 2048), (512, 1024, 4096), (1000, 1024, 4096), (1531, 1024, 3584), (2048, 1024, 4096),
                (2048, 1024, 14336), (2048, 1024, 16384)):
    int8(t, k, n)
for t, v, n in ((1, 50000, 5), (2000, 300, 5)):
    logprobs(t, v, n)
torch.cuda.synchronize()
graphs = []
for name, outs, call in calls:
    print("record", name, flush=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    graphs.append(graph)
for (name, outs, call), graph in zip(calls, graphs):
    print("replay", name, flush=True)
    got = []
    for _ in range(3):
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got.append([o.clone() for o in outs])
    for o in outs:
        o.zero_()
    call()
    torch.cuda.synchronize()
    for replay in got:
        assert all(torch.equal(a, b) for a, b in zip(replay, outs)), name
        assert all(a.float().abs().sum() > 0 for a in replay[:1]), name
print("all the same")
"""


@pytest.mark.gpu
def test_first_calls_may_be_recorded():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-u", "-c", CHILD], cwd=root, capture_output=True, text=True, timeout=100)
    assert run.returncode == 0 and run.stdout.endswith("all the same\n"), run.stdout[-500:] + run.stderr[-2000:]
