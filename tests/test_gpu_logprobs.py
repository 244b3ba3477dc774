"""rsllm_hip_token_logprobs_dev against 64-bit arithmetic: ids and ranks equal,
log-probabilities and entropies within the f32 roundings of the formula."""
import numpy as np
import pytest
import torch

import serving_ref as R

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")
U = 2.0 ** -24


def bounds(values, lp, ent, top):
    """What the roundings can add up to. exp of x = l - m is off by (|x| + 3) U
    relative (x rounded, its product with log2 e rounded, the exponential's own
    step); a chain of at most v / 256 + 64 additions adds as many U; so does the
    second sum, relative to sum e |x|. log S then carries that error, and x, log S
    and their difference are rounded once each."""
    out = []
    for t, l in enumerate(values):
        live = l[l > -np.inf]
        with np.errstate(all="ignore"):
            m = live.max() if live.size else 0.0
            x = np.where(live == m, 0.0, live - m)
            e = np.exp(x)
            mean = (e * np.abs(np.where(e > 0, x, 0))).sum() / max(e.sum(), 1e-300)
            log_s = np.log(max(e.sum(), 1.0))
        chain = len(l) / 256 + 64
        rel = (chain + mean + 4) * U
        out.append((rel + 2 * log_s * U, (rel + 2 * U) * (1 + 3 * mean) + 3 * (log_s + mean) * U
                    + 30 * mean * U))
    a, b = (np.array(v) for v in zip(*out))
    with np.errstate(invalid="ignore"):
        return (a + 3 * U * np.abs(np.nan_to_num(lp, posinf=0, neginf=0)), b,
                a[:, None] + 3 * U * np.abs(np.nan_to_num(top, posinf=0, neginf=0)))


def near(got, want, bound):
    got = got.astype(np.float64)
    want = np.where(np.abs(want) > 3.4028236e38, np.copysign(INF, want), want)  # f32's largest
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    with np.errstate(invalid="ignore"):
        ok = same | (np.abs(got - want) <= bound)
    assert ok.all(), (got[~ok][:5], want[~ok][:5], np.broadcast_to(bound, want.shape)[~ok][:5])


def run(hip, logits, tokens, n_top, dtype="f32", stride=None, offset=0, stream=None, skip=()):
    t, values = R.as_type(logits, dtype)
    n_tok, v = t.shape
    buf, span = R.strided(t, stride or v)
    store = torch.full((offset + buf.numel(),), NAN, dtype=buf.dtype)
    store[offset:] = buf.reshape(-1)
    d = store.cuda()
    tok = None if tokens is None else torch.tensor(tokens, dtype=torch.int32, device="cuda")
    f = torch.full((2, n_tok + 4), -7.0, device="cuda")
    rank = torch.full((n_tok + 4,), -7, dtype=torch.int32, device="cuda")
    ids = torch.full((n_tok * n_top + 4,), -7, dtype=torch.int32, device="cuda")
    top = torch.full((n_tok * n_top + 4,), -7.0, device="cuda")
    work = torch.full((hip.token_logprobs_work_bytes(n_tok, v, n_top) + 256,), 0xCD, dtype=torch.uint8,
                      device="cuda")
    torch.cuda.synchronize()
    hip.token_logprobs_dev(f[0].data_ptr() if tokens is not None else 0,
                           0 if "entropy" in skip else f[1].data_ptr(),
                           0 if "rank" in skip or tokens is None else rank.data_ptr(), n_tok,
                           ids.data_ptr() if n_top else 0, top.data_ptr() if n_top else 0,
                           n_tok * n_top, d.data_ptr() + offset * d.element_size(), span, stride or v,
                           0 if tok is None else tok.data_ptr(), 0 if tok is None else n_tok,
                           work.data_ptr(), work.numel(), n_tok, v, n_top, R.GGML[dtype],
                           stream or torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert (work[-256:] == 0xCD).all(), "wrote behind the workspace"
    f, rank, ids, top = (a.cpu().numpy() for a in (f, rank, ids, top))
    for a in (f[0, n_tok:], f[1, n_tok:], rank[n_tok:], ids[n_tok * n_top:], top[n_tok * n_top:]):
        assert (a == -7).all(), "wrote behind an output"
    lp, want_rank, ent, want_ids, want_top = R.logprobs(values, tokens, n_top)
    b_lp, b_ent, b_top = bounds(values, lp, ent, want_top)
    np.testing.assert_array_equal(ids[:n_tok * n_top].reshape(n_tok, n_top), want_ids)
    near(top[:n_tok * n_top].reshape(n_tok, n_top), want_top, b_top)
    if tokens is None:
        assert (f[0] == -7).all() and (rank == -7).all()
    else:
        near(f[0, :n_tok], lp, b_lp)
        if "rank" in skip:
            assert (rank == -7).all()
        else:
            np.testing.assert_array_equal(rank[:n_tok], want_rank)
    if "entropy" in skip:
        assert (f[1] == -7).all()
    else:
        near(f[1, :n_tok], ent, b_ent)


def model_logits(rng, n_tok, v):
    x = rng.normal(0, 2.5, (n_tok, v))
    tok = rng.integers(0, v, n_tok)
    x[np.arange(n_tok), tok] += 8
    return x, tok.tolist()


@pytest.mark.parametrize("n_tok,v,n_top", [
    (1, 1, 1), (1, 1, 0), (2, 3, 3), (1, 63, 5), (3, 64, 64), (5, 65, 64), (2, 255, 20), (1, 257, 1),
    (4, 1000, 5), (1, 4095, 20), (1, 4097, 64), (2, 8193, 8), (1, 32000, 20), (3, 50257, 64),
    (1, 129280, 8), (2, 129280, 64), (1, 200001, 5), (40, 5000, 3), (300, 2000, 5), (520, 1024, 20),
    (1100, 333, 1), (17, 31999, 0)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_sizes(hip, dtype, n_tok, v, n_top):
    rng = np.random.default_rng(n_tok * v)
    x, tok = model_logits(rng, n_tok, v)
    run(hip, x, tok, n_top, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("stride,offset", [(1000, 0), (1001, 0), (1003, 1), (1008, 3), (1000, 5), (1024, 7)])
def test_strides_and_starts(hip, dtype, stride, offset):
    rng = np.random.default_rng(stride + offset)
    x, tok = model_logits(rng, 9, 1000)
    run(hip, x, tok, 10, dtype, stride, offset)


def test_optional_outputs(hip):
    rng = np.random.default_rng(2)
    x, tok = model_logits(rng, 3, 3001)
    run(hip, x, tok, 5, skip=("rank",))
    run(hip, x, tok, 5, skip=("entropy",))
    run(hip, x, None, 5)
    run(hip, x, None, 0)
    run(hip, x, tok, 0, skip=("rank", "entropy"))


@pytest.mark.parametrize("v", [700, 9000, 140000])
def test_equal_logits(hip, v):
    """Whole rows of one value, few values, and the largest ones far apart: equal
    logits in rising order of id."""
    rng = np.random.default_rng(v)
    x = np.zeros((5, v))
    x[1] = rng.integers(0, 3, v)
    x[2, ::97] = 1.0
    x[3, [v - 1, v // 2, 3]] = 2.0
    x[4, ::2] = -0.0
    run(hip, x, [0, 5, 97, v - 1, 1], 20)
    run(hip, x, [0, 5, 97, v - 1, 1], 64, "bf16")


@pytest.mark.parametrize("v", [700, 9000, 30000])
def test_ordered_rows(hip, v):
    """Rising and falling logits: every one, or none, is a new largest."""
    x = np.stack([np.linspace(-20, 20, v), np.linspace(20, -20, v),
                  np.abs(np.linspace(-20, 20, v)), np.r_[np.linspace(-9, 9, v - v // 2), np.full(v // 2, -3.0)]])
    run(hip, x, [0, 0, v // 2, v - 1], 20)
    run(hip, x, [v - 1, v - 1, 0, 5], 64, "f16")


@pytest.mark.parametrize("v", [130, 5000, 70001])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_masked_rows(hip, v, dtype):
    """-inf: probability 0 and never listed; rows with three, one and no tokens
    left, and a given token that is masked."""
    rng = np.random.default_rng(v)
    x, tok = model_logits(rng, 8, v)
    x[0] = np.where(rng.random(v) < 0.9, -INF, x[0])
    x[1] = -INF
    x[2] = -INF
    x[2, [3, v // 2, v - 1]] = [1.0, 2.0, 1.0]
    x[3] = -INF
    x[3, 77] = -5.0
    x[4, tok[4]] = -INF
    x[5, :v // 2] = -INF
    x[6, v // 2:] = -INF
    x[7] = np.float32(-3.0e38)
    run(hip, x, tok, 8, dtype)
    tok[3] = 77
    run(hip, x, tok, 20, dtype)


@pytest.mark.parametrize("v", [130, 5000, 70001])
def test_infinities_and_nan(hip, v):
    rng = np.random.default_rng(v)
    x, tok = model_logits(rng, 6, v)
    x[0, 9] = INF
    x[1, [9, v - 2]] = INF
    x[2, v - 1] = NAN
    x[3, tok[3]] = NAN
    x[4] = NAN
    tok[1] = 9
    x[5] = np.r_[np.full(v - 1, -3e38), 3e38]  # differences beyond f32's range
    run(hip, x, tok, 8)


def test_tokens_outside_the_vocabulary(hip):
    rng = np.random.default_rng(4)
    x, _ = model_logits(rng, 5, 900)
    run(hip, x, [-1, 900, 2 ** 31 - 1, -2 ** 31, 899], 3)


def test_large_logits_and_long_rows(hip):
    rng = np.random.default_rng(5)
    x = rng.normal(0, 1, (2, 100000))
    run(hip, x * 1e4, [5, 6], 8)
    run(hip, x * 1e-6, [5, 6], 8)  # all but uniform: entropy near log v
    run(hip, np.zeros((1, 250000)) + 30000.0, [9], 4)


def test_on_another_stream_and_captured(hip):
    rng = np.random.default_rng(6)
    x, tok = model_logits(rng, 3, 20000)
    side = torch.cuda.Stream()
    run(hip, x, tok, 8, stream=side.cuda_stream)
    graphs, before = [], hip.device_allocations()
    for n_tok in (1, 40):
        d = torch.zeros(n_tok, 20000, device="cuda")
        t = torch.zeros(n_tok, dtype=torch.int32, device="cuda")
        o = torch.zeros(2, n_tok, device="cuda")
        rank = torch.zeros(n_tok, dtype=torch.int32, device="cuda")
        ids = torch.zeros(n_tok, 8, dtype=torch.int32, device="cuda")
        top = torch.zeros(n_tok, 8, device="cuda")
        work = torch.empty(max(256, hip.token_logprobs_work_bytes(n_tok, 20000, 8)), dtype=torch.uint8,
                           device="cuda")
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            hip.token_logprobs_dev(o[0].data_ptr(), o[1].data_ptr(), rank.data_ptr(), n_tok,
                                   ids.data_ptr(), top.data_ptr(), n_tok * 8, d.data_ptr(), d.numel(),
                                   20000, t.data_ptr(), n_tok, work.data_ptr(), work.numel(), n_tok,
                                   20000, 8, stream=torch.cuda.current_stream().cuda_stream)
        graphs.append((n_tok, d, t, o, rank, ids, top, work, g, torch.cuda.Stream()))
    assert hip.device_allocations() == before
    for i in range(4):
        want = []
        for n_tok, d, t, o, *_ in graphs:
            x, tok = model_logits(rng, n_tok, 20000)
            x = x.astype(np.float32)
            d.copy_(torch.from_numpy(x))
            t.copy_(torch.tensor(tok, dtype=torch.int32))
            o.fill_(NAN)
            want.append((x.astype(np.float64), R.logprobs(x.astype(np.float64), tok, 8)))
        torch.cuda.synchronize()
        for entry in graphs:
            with torch.cuda.stream(entry[-1]):
                entry[-2].replay()
        torch.cuda.synchronize()
        for (n_tok, d, t, o, rank, ids, top, *_), (x, (lp, r, ent, want_ids, want_top)) in zip(graphs, want):
            b_lp, b_ent, b_top = bounds(x, lp, ent, want_top)
            near(o[0].cpu().numpy(), lp, b_lp)
            near(o[1].cpu().numpy(), ent, b_ent)
            near(top.cpu().numpy(), want_top, b_top)
            np.testing.assert_array_equal(rank.cpu().numpy(), r)
            np.testing.assert_array_equal(ids.cpu().numpy(), want_ids)


def test_rows_beyond_32_bit_offsets(hip):
    """4.7 GB of logits: the first and the last rows."""
    n_tok, v = 9100, 129280
    d = torch.randn(n_tok, v, device="cuda")
    tok = torch.randint(0, v, (n_tok,), dtype=torch.int32, device="cuda")
    o, rank = torch.full((2, n_tok), NAN, device="cuda"), torch.zeros(n_tok, dtype=torch.int32, device="cuda")
    ids, top = torch.zeros(n_tok, 5, dtype=torch.int32, device="cuda"), torch.zeros(n_tok, 5, device="cuda")
    work = torch.empty(256 + hip.token_logprobs_work_bytes(n_tok, v, 5), dtype=torch.uint8, device="cuda")
    hip.token_logprobs_dev(o[0].data_ptr(), o[1].data_ptr(), rank.data_ptr(), n_tok, ids.data_ptr(),
                           top.data_ptr(), n_tok * 5, d.data_ptr(), d.numel(), v, tok.data_ptr(), n_tok,
                           work.data_ptr(), work.numel(), n_tok, v, 5,
                           stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    for at in (slice(0, 2), slice(n_tok - 2, n_tok)):
        x = d[at].cpu().double().numpy()
        lp, r, ent, want_ids, want_top = R.logprobs(x, tok[at].cpu().tolist(), 5)
        b_lp, b_ent, b_top = bounds(x, lp, ent, want_top)
        near(o[0, at].cpu().numpy(), lp, b_lp)
        near(o[1, at].cpu().numpy(), ent, b_ent)
        near(top[at].cpu().numpy(), want_top, b_top)
        np.testing.assert_array_equal(rank[at].cpu().numpy(), r)
        np.testing.assert_array_equal(ids[at].cpu().numpy(), want_ids)


@pytest.mark.parametrize("parts", [2, 3, 7, 8, 9])
def test_lists_of_parts(hip, parts):
    """Rows cut into a few parts, lists as long as their number, one longer and 64
    long: the best in one part, in its first or last, masked parts, equal logits
    across parts."""
    v = 4096 * parts - 40
    rng = np.random.default_rng(parts)
    x, tok = model_logits(rng, 6, v)
    x[1, v - 100:] += 40.0
    x[2, :100] += 40.0
    x[3, 4000:] = -INF
    x[4, :v - 5] = -INF
    x[5] = rng.integers(0, 2, v)
    for n_top in (parts, parts + 1, 64):
        run(hip, x, tok, n_top)
