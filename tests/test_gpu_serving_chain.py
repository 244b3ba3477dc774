"""A token's way through the routing, the routed experts, the int8 product and
the log-probabilities, as a serving loop enqueues it: one stream, no host
synchronisation, then captured into a graph and replayed. Every stage is checked
on what the stage before it wrote."""
import numpy as np
import pytest
import torch

import serving_ref as R
from conftest import REL_TOL, rel_err
from rsllm_amd import synth
from rsllm_amd.ggml import GgmlType as G
from test_gpu_logprobs import bounds, near

pytestmark = pytest.mark.gpu

EMBD, FF, EXPERTS, TOP, VOCAB, N_TOP = 1024, 512, 32, 4, 5003, 6


class Chain:
    def __init__(self, hip, n_tok, seed):
        rng = np.random.default_rng(seed)
        self.hip, self.t = hip, n_tok
        self.gate, self.up = (synth.weight(G.Q4_K, EXPERTS * FF, EMBD, seed + i) for i in (1, 2))
        self.down = synth.weight(G.Q4_K, EXPERTS * EMBD, FF, seed + 3)
        self.router = (rng.normal(0, 1.5, (EXPERTS, EMBD)) / EMBD ** 0.5).astype(np.float32)
        self.bias = rng.normal(0, 0.05, EXPERTS).astype(np.float32)
        head = torch.from_numpy(rng.normal(0, 1, (VOCAB, EMBD)).astype(np.float32)).cuda()

        def new(*shape, dtype=torch.float32):
            return torch.zeros(*shape, dtype=dtype, device="cuda")
        self.d = {k: torch.from_numpy(getattr(self, k)).cuda() for k in ("gate", "up", "down", "router", "bias")}
        # the head's channels are quantised by the same call as tokens are
        self.w, self.ws = new(VOCAB, hip.int8_row_bytes(EMBD), dtype=torch.int8), new(VOCAB)
        hip.quantize_int8_dev(head.data_ptr(), head.numel(), EMBD, self.w.data_ptr(), self.w.numel(),
                              self.ws.data_ptr(), VOCAB, VOCAB, EMBD, G.F32,
                              torch.cuda.current_stream().cuda_stream)
        self.x, self.h = new(n_tok, EMBD), new(n_tok, EMBD)
        self.router_logits = new(n_tok, EXPERTS)
        self.ids, self.wts = new(n_tok, TOP, dtype=torch.int32), new(n_tok, TOP)
        self.logits = new(n_tok, VOCAB, dtype=torch.bfloat16)
        self.tokens = new(n_tok, dtype=torch.int32)
        self.lp, self.ent, self.rank = new(n_tok), new(n_tok), new(n_tok, dtype=torch.int32)
        self.top_ids, self.top = new(n_tok, N_TOP, dtype=torch.int32), new(n_tok, N_TOP)
        self.work = new(hip.int8_work_bytes(n_tok, EMBD, VOCAB), dtype=torch.uint8)
        self.work2 = new(256 + hip.token_logprobs_work_bytes(n_tok, VOCAB, N_TOP), dtype=torch.uint8)
        torch.cuda.synchronize()

    def load(self, seed):
        rng = np.random.default_rng(seed)
        self.x.copy_(torch.from_numpy(rng.normal(0, 1, (self.t, EMBD)).astype(np.float32)))
        self.tokens.copy_(torch.from_numpy(rng.integers(0, VOCAB, self.t).astype(np.int32)))

    def enqueue(self):
        hip, t, d = self.hip, self.t, self.d
        st = torch.cuda.current_stream().cuda_stream
        hip.matmul_weight_f32_dev(self.router_logits.data_ptr(), t * EXPERTS, d["router"].data_ptr(),
                                  EXPERTS * EMBD * 4, self.x.data_ptr(), t * EMBD, t, EMBD, EXPERTS, G.F32, st)
        hip.moe_route_dev(self.ids.data_ptr(), self.wts.data_ptr(), t * TOP, self.router_logits.data_ptr(),
                          t * EXPERTS, EXPERTS, d["bias"].data_ptr(), EXPERTS, t, EXPERTS, TOP, 4, 2, 2,
                          hip.RouteScore.SqrtSoftplus, True, 1.5, G.F32, st)
        self.h.copy_(self.x)  # the experts add to the residual
        hip.moe_routed_dev(self.h.data_ptr(), t * EMBD, self.x.data_ptr(), t * EMBD, d["gate"].data_ptr(),
                           d["up"].data_ptr(), d["gate"].numel(), d["down"].data_ptr(), d["down"].numel(),
                           self.ids.data_ptr(), self.wts.data_ptr(), t * TOP, t, EMBD, FF, EXPERTS, TOP,
                           G.Q4_K, G.Q4_K, 10.0, st)
        hip.matmul_int8_dev(self.logits.data_ptr(), t * VOCAB, VOCAB, self.w.data_ptr(), self.w.numel(),
                            self.ws.data_ptr(), VOCAB, 0, 0, self.h.data_ptr(), t * EMBD, EMBD,
                            self.work.data_ptr(), self.work.numel(), t, EMBD, VOCAB, G.F32, G.BF16, st)
        hip.token_logprobs_dev(self.lp.data_ptr(), self.ent.data_ptr(), self.rank.data_ptr(), t,
                               self.top_ids.data_ptr(), self.top.data_ptr(), t * N_TOP,
                               self.logits.data_ptr(), t * VOCAB, VOCAB, self.tokens.data_ptr(), t,
                               self.work2.data_ptr(), self.work2.numel(), t, VOCAB, N_TOP, G.BF16, st)

    def outputs(self):
        return [a.clone() for a in (self.ids, self.wts, self.h, self.logits, self.lp, self.ent, self.rank,
                                    self.top_ids, self.top)]

    def check(self, oracle):
        t = self.t

        def f64(a):
            return a.cpu().double().numpy()
        x = self.x.cpu().numpy()
        want = x.astype(np.float64) @ self.router.astype(np.float64).T
        assert rel_err(self.router_logits.cpu().numpy(), want) <= REL_TOL
        ids, wts = R.route(f64(self.router_logits), self.bias.astype(np.float64), TOP, 4, 2, 2, 2, True, 1.5)
        np.testing.assert_array_equal(self.ids.cpu().numpy(), ids)
        np.testing.assert_allclose(f64(self.wts), wts, rtol=2.0 ** -23)
        h = x.reshape(-1).copy()
        assert oracle.moe_routed(h, x.reshape(-1), t, EMBD, FF, self.gate, self.up, self.down, int(G.Q4_K),
                                 int(G.Q4_K), EXPERTS, self.ids.cpu().numpy().reshape(-1),
                                 self.wts.cpu().numpy().reshape(-1), TOP, 10.0) == 0
        assert rel_err(self.h.cpu().numpy().reshape(-1), h) <= REL_TOL
        codes, scales = R.quantize(f64(self.h))
        y, p = R.int8_product(codes, scales, self.w[:, :EMBD].cpu().numpy(), self.ws.cpu().numpy(), None)
        bound = 3.001 * 2.0 ** -24 * np.abs(p) + 1.001 * R.HALF_STEP["bf16"] * np.abs(y) + R.TINY_STEP["bf16"]
        assert not (np.abs(f64(self.logits) - y) > bound).any()
        logits = f64(self.logits)
        lp, rank, ent, top_ids, top = R.logprobs(logits, self.tokens.cpu().tolist(), N_TOP)
        b_lp, b_ent, b_top = bounds(logits, lp, ent, top)
        near(self.lp.cpu().numpy(), lp, b_lp)
        near(self.ent.cpu().numpy(), ent, b_ent)
        near(self.top.cpu().numpy(), top, b_top)
        np.testing.assert_array_equal(self.rank.cpu().numpy(), rank)
        np.testing.assert_array_equal(self.top_ids.cpu().numpy(), top_ids)


@pytest.mark.parametrize("n_tok", [1, 5, 40])
def test_chain_eager_and_captured(hip, oracle, n_tok):
    hip.init(0)
    c = Chain(hip, n_tok, 7000 + n_tok)
    c.load(1)
    c.enqueue()
    torch.cuda.synchronize()
    c.check(oracle)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):  # the routed experts make this stream's workspace
        c.enqueue()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        c.enqueue()
    for seed in (2, 3, 4):
        c.load(seed)
        torch.cuda.synchronize()
        c.enqueue()
        torch.cuda.synchronize()
        eager = c.outputs()
        c.lp.fill_(float("nan"))
        c.ids.fill_(-9)
        c.logits.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager, c.outputs()):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    c.check(oracle)
    hip.stream_release(side.cuda_stream)
