"""The 4-bit calls one behind another, as a model's step uses them: weights quantised on the
GPU, a layer's experts, an FFN's gate and up products on activations quantised once, the
head, and the log-probabilities of its logits; each step against 64-bit arithmetic of what it
was given, and the whole captured and replayed."""
import numpy as np
import pytest
import torch

import mxfp4_ref as M
import serving_ref as R
from test_gpu_logprobs import bounds, near
from test_gpu_mxfp4 import dev

pytestmark = pytest.mark.gpu

EMBD, FF, EXPERTS, TOP, VOCAB, N_TOP = 320, 144, 12, 3, 1030, 5
F32, BF16 = 0, 30


class Step:
    def __init__(self, hip, t):
        self.hip, self.t = hip, t
        rng = np.random.default_rng(t)
        self.router = (rng.normal(0, 1.5, (EXPERTS, EMBD)) / np.sqrt(EMBD)).astype(np.float32)
        all_ = EXPERTS + 1
        self.m = {}
        for name, rows, k in (("gate", all_ * FF, EMBD), ("up", all_ * FF, EMBD), ("down", all_ * EMBD, FF),
                              ("g2", FF, EMBD), ("u2", FF, EMBD), ("head", VOCAB, EMBD)):
            w = torch.from_numpy(rng.normal(0, 2.0 / np.sqrt(k), (rows, k))).to(torch.bfloat16)
            self.m[name] = (w, *self.quantised(w.cuda(), BF16))
        self.d = {"router": dev(self.router)}
        u8 = dict(dtype=torch.uint8, device="cuda")
        self.x = torch.zeros(t, EMBD, device="cuda")
        self.h = torch.zeros(t, EMBD, dtype=torch.bfloat16, device="cuda")
        self.ids = torch.zeros(t, TOP, dtype=torch.int32, device="cuda")
        self.wts = torch.zeros(t, TOP, device="cuda")
        self.codes = torch.zeros(t, M.row_bytes(EMBD), **u8)
        self.scales = torch.zeros(t, M.scale_bytes(EMBD), **u8)
        self.g2, self.u2 = (torch.zeros(t, FF, device="cuda") for _ in range(2))
        self.logits = torch.zeros(t, VOCAB, device="cuda")
        self.tokens = torch.zeros(t, dtype=torch.int32, device="cuda")
        self.lp, self.ent = torch.zeros(t, device="cuda"), torch.zeros(t, device="cuda")
        self.rank = torch.zeros(t, dtype=torch.int32, device="cuda")
        self.top_ids = torch.zeros(t, N_TOP, dtype=torch.int32, device="cuda")
        self.top = torch.zeros(t, N_TOP, device="cuda")
        g, u, w = (self.m[k] for k in ("gate", "up", "down"))
        self.layer = hip.MoeMxfp4(
            router=self.d["router"].data_ptr(), router_len=EXPERTS * EMBD, dtype_router=F32, bias=0, bias_len=0,
            gate=g[1].data_ptr(), up=u[1].data_ptr(), gate_up_len=g[1].numel(), gate_scales=g[2].data_ptr(),
            up_scales=u[2].data_ptr(), gate_up_scales_len=g[2].numel(), down=w[1].data_ptr(), down_len=w[1].numel(),
            down_scales=w[2].data_ptr(), down_scales_len=w[2].numel(), n_embd=EMBD, n_ff=FF, n_expert=EXPERTS,
            n_shared=1, k=TOP, n_group=1, topk_group=1, group_top=1, score=2, renormalise=1, scale=1.5, clamp=10.0)
        # one workspace, which the calls use one after the other
        self.work = torch.empty(max(1, hip.moe_mxfp4_work_bytes(self.layer, t), hip.mxfp4_work_bytes(t, EMBD, FF),
                                    hip.mxfp4_work_bytes(t, EMBD, VOCAB),
                                    hip.token_logprobs_work_bytes(t, VOCAB, N_TOP)), **u8)

    def quantised(self, x, kind):
        n, k = x.shape
        codes = torch.empty(n, M.row_bytes(k), dtype=torch.uint8, device="cuda")
        scales = torch.empty(n, M.scale_bytes(k), dtype=torch.uint8, device="cuda")
        self.hip.quantize_mxfp4_dev(x.data_ptr(), x.numel(), k, codes.data_ptr(), codes.numel(), scales.data_ptr(),
                                    scales.numel(), n, k, kind, torch.cuda.current_stream().cuda_stream)
        return codes, scales

    def inputs(self, seed):
        rng = np.random.default_rng(seed)
        self.x.copy_(torch.from_numpy(rng.normal(0, 1, (self.t, EMBD)).astype(np.float32)))
        self.tokens.copy_(torch.from_numpy(rng.integers(0, VOCAB, self.t).astype(np.int32)))

    def enqueue(self):
        hip, t = self.hip, self.t
        st = torch.cuda.current_stream().cuda_stream
        work = (self.work.data_ptr(), self.work.numel())
        hip.moe_mxfp4_dev(self.layer, self.h.data_ptr(), t * EMBD, EMBD, self.ids.data_ptr(), self.wts.data_ptr(),
                          t * TOP, self.x.data_ptr(), t * EMBD, EMBD, *work, t, F32, BF16, st)
        hip.quantize_mxfp4_dev(self.h.data_ptr(), t * EMBD, EMBD, self.codes.data_ptr(), self.codes.numel(),
                               self.scales.data_ptr(), self.scales.numel(), t, EMBD, BF16, st)
        for name, out in (("g2", self.g2), ("u2", self.u2)):
            _, w, ws = self.m[name]
            hip.matmul_mxfp4_prequant_dev(out.data_ptr(), t * FF, FF, w.data_ptr(), w.numel(), ws.data_ptr(),
                                          ws.numel(), 0, 0, self.codes.data_ptr(), self.codes.numel(),
                                          self.scales.data_ptr(), self.scales.numel(), *work, t, EMBD, FF, F32, st)
        _, w, ws = self.m["head"]
        hip.matmul_mxfp4_dev(self.logits.data_ptr(), t * VOCAB, VOCAB, w.data_ptr(), w.numel(), ws.data_ptr(),
                             ws.numel(), 0, 0, self.h.data_ptr(), t * EMBD, EMBD, *work, t, EMBD, VOCAB, BF16, F32, st)
        hip.token_logprobs_dev(self.lp.data_ptr(), self.ent.data_ptr(), self.rank.data_ptr(), t,
                               self.top_ids.data_ptr(), self.top.data_ptr(), t * N_TOP, self.logits.data_ptr(),
                               t * VOCAB, VOCAB, self.tokens.data_ptr(), t, *work, t, VOCAB, N_TOP, F32, st)

    def outputs(self):
        return [a.clone() for a in (self.ids, self.wts, self.h, self.codes, self.scales, self.g2, self.u2, self.logits,
                                    self.lp, self.ent, self.rank, self.top_ids, self.top)]

    def check(self):
        def f64(a):
            return a.cpu().double().numpy()
        v = {}
        for name, (w, codes, scales) in self.m.items():
            want = M.quantize(f64(w[:64]))  # (a part of the rows: the plain form is slow)
            assert np.array_equal(codes[:64].cpu().numpy(), want[0])
            assert np.array_equal(scales[:64].cpu().numpy(), want[1])
            v[name] = M.values(codes.cpu().numpy(), scales.cpu().numpy(), w.shape[1])
        ids, wts, h, tol = M.moe(f64(self.x), self.router.astype(np.float64), None, v["gate"].reshape(-1, FF, EMBD),
                                 v["up"].reshape(-1, FF, EMBD), v["down"].reshape(-1, EMBD, FF), EXPERTS, 1, TOP, 1, 1,
                                 1, 2, True, 1.5, 10.0, "bf16")
        np.testing.assert_array_equal(self.ids.cpu().numpy(), ids)
        np.testing.assert_allclose(f64(self.wts), wts, rtol=2.0 ** -23)
        assert (np.abs(f64(self.h) - h) <= tol).all()
        codes, scales = M.quantize(f64(self.h))
        assert np.array_equal(self.codes.cpu().numpy(), codes) and np.array_equal(self.scales.cpu().numpy(), scales)
        q = M.values(codes, scales, EMBD)
        for name, out in (("g2", self.g2), ("u2", self.u2), ("head", self.logits)):
            y, size = M.product(q, v[name], None)
            bound = ((EMBD + 127) // 128 + 17) * 2.0 ** -23 * size + M.rounding(y, "f32")
            assert (np.abs(f64(out) - y) <= bound).all()
        logits = f64(self.logits)
        lp, rank, ent, top_ids, top = R.logprobs(logits, self.tokens.cpu().tolist(), N_TOP)
        b_lp, b_ent, b_top = bounds(logits, lp, ent, top)
        near(self.lp.cpu().numpy(), lp, b_lp)
        near(self.ent.cpu().numpy(), ent, b_ent)
        near(self.top.cpu().numpy(), top, b_top)
        np.testing.assert_array_equal(self.rank.cpu().numpy(), rank)
        np.testing.assert_array_equal(self.top_ids.cpu().numpy(), top_ids)


@pytest.mark.parametrize("t", [1, 7, 32])
def test_chain_eager_and_captured(hip, t):
    s = Step(hip, t)
    s.inputs(0)
    before = hip.device_allocations()
    s.enqueue()
    s.check()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        s.enqueue()
    for i in range(1, 4):
        s.inputs(i)
        s.work.random_(0, 256)
        graph.replay()
        torch.cuda.synchronize()
        s.check()
        replayed = s.outputs()
        for a in (s.h, s.codes, s.scales, s.logits, s.lp):
            a.zero_()
        s.enqueue()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(replayed, s.outputs()))
    assert hip.device_allocations() == before
