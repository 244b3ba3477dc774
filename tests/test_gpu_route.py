"""rsllm_hip_moe_route_dev against a 64-bit implementation: ids equal, weights
within the one rounding to f32."""
import numpy as np
import pytest
import torch

import serving_ref as R

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def run(hip, logits, bias, k, n_group=1, topk_group=1, group_top=1, score=0, renorm=True,
        scale=1.0, dtype="f32", stride=None, stream=None, offset=0):
    t, values = R.as_type(logits, dtype)
    n_tok, n = t.shape
    buf, span = R.strided(t, stride or n)
    # the rows start `offset` elements into the allocation
    store = torch.full((offset + buf.numel(),), NAN, dtype=buf.dtype)
    store[offset:] = buf.reshape(-1)
    d = store.cuda()
    b = None if bias is None else torch.from_numpy(np.asarray(bias, np.float32)).cuda()
    ids = torch.full((n_tok * k + 8,), -77, dtype=torch.int32, device="cuda")
    w = torch.full((n_tok * k + 8,), -77.0, device="cuda")
    torch.cuda.synchronize()
    hip.moe_route_dev(ids.data_ptr(), w.data_ptr(), n_tok * k,
                      d.data_ptr() + offset * d.element_size(), span, stride or n,
                      0 if b is None else b.data_ptr(), 0 if b is None else n, n_tok, n, k, n_group,
                      topk_group, group_top, score, renorm, scale, R.GGML[dtype],
                      stream or torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    ids, w = ids.cpu().numpy(), w.cpu().numpy()
    assert (ids[n_tok * k:] == -77).all() and (w[n_tok * k:] == -77).all()
    bias64 = None if bias is None else np.asarray(bias, np.float32).astype(np.float64)
    want_ids, want_w = R.route(values, bias64, k, n_group, topk_group, group_top, score, renorm, scale)
    ids, w = ids[:n_tok * k].reshape(n_tok, k), w[:n_tok * k].reshape(n_tok, k)
    np.testing.assert_array_equal(ids, want_ids)
    # 64-bit arithmetic throughout, then one rounding to f32
    np.testing.assert_allclose(w.astype(np.float64), want_w, rtol=2.0 ** -24 * (1 + 1e-6),
                               atol=2.0 ** -150)
    return ids, w


@pytest.mark.parametrize("score", [0, 1, 2])
@pytest.mark.parametrize("n_tok,n,k,groups", [
    (1, 1, 1, (1, 1, 1)), (1, 256, 8, (8, 4, 2)), (3, 8, 2, (1, 1, 1)), (33, 60, 4, (1, 1, 1)),
    (5, 63, 63, (1, 1, 1)), (5, 65, 64, (1, 1, 1)), (17, 160, 6, (8, 3, 1)), (65, 256, 6, (1, 1, 1)),
    (9, 384, 8, (1, 1, 1)), (4, 513, 10, (1, 1, 1)), (3, 1000, 12, (4, 2, 2)),
    (2, 2000, 7, (1, 1, 1)), (2, 4096, 16, (16, 5, 2)), (1, 16384, 64, (1024, 100, 2)),
    (7, 128, 4, (128, 5, 2)), (7, 96, 24, (4, 1, 2)),
])
def test_sizes(hip, score, n_tok, n, k, groups):
    rng = np.random.default_rng(n * 7 + k + score)
    x = rng.normal(0, 1.5, (n_tok, n))
    run(hip, x, rng.normal(0, 0.05, n), k, *groups, score=score, scale=2.5)
    run(hip, x, None, k, *groups, score=score, renorm=False)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("stride,offset", [(None, 0), (67, 0), (130, 1), (64, 3)])
def test_types_strides_and_starts(hip, dtype, stride, offset):
    rng = np.random.default_rng(5)
    run(hip, rng.normal(0, 1.5, (21, 64)), rng.normal(0, 0.05, 64), 6, 4, 2, 2, score=1,
        dtype=dtype, stride=stride, offset=offset)
    run(hip, rng.normal(0, 1.5, (21, 64)), None, 6, dtype=dtype, stride=stride, offset=offset)


@pytest.mark.parametrize("score", [0, 1, 2])
@pytest.mark.parametrize("bias", [False, True])
def test_equal_places_go_to_the_lower_id(hip, score, bias):
    rng = np.random.default_rng(6)
    x = rng.integers(-2, 3, (40, 256)).astype(np.float64)
    x[0] = 0.0
    x[1, ::2] = -0.0  # one place with 0
    x[1, 1::2] = 0.0
    run(hip, x, np.full(256, 0.25) if bias else None, 8, score=score)
    run(hip, x, np.full(256, 0.25) if bias else None, 8, 8, 4, 2, score=score)


def test_keys_that_differ_by_less_than_a_32_bit_rounding(hip):
    """Scores near 1 whose difference f32 does not hold: the order is the 64-bit
    one."""
    x = np.full((2, 128), 15.0, np.float32)
    x[0] = np.nextafter(np.float32(15.0), np.float32(99), dtype=np.float32)
    x[0, 5:9] = 15.0
    x[1, 77] = np.nextafter(np.float32(15.0), np.float32(99), dtype=np.float32)
    bias = np.zeros(128)
    bias[64:] = 0.0
    ids, _ = run(hip, x, bias, 4, score=1)
    assert ids[1, 0] == 77


@pytest.mark.parametrize("score", [0, 1, 2])
@pytest.mark.parametrize("groups", [(1, 1, 1), (8, 4, 2), (8, 4, 1)])
@pytest.mark.parametrize("n,k", [(64, 8), (256, 8), (256, 20), (384, 8), (1000, 64)])
def test_close_keys(hip, score, groups, n, k):
    """Rows whose logits are a few f32 steps apart, and rows of few values among
    which such pairs are: neighbours in the order, the last chosen and the first
    left out, and groups are settled by the 64-bit keys."""
    rng = np.random.default_rng(n + k + score)
    step = np.float32(2.0 ** -23)
    rows = []
    for base in (1.0, -1.5, 3.0):
        rows.append(np.float32(base) + step * rng.integers(0, 40, n).astype(np.float32) * 2)
        rows.append(np.float32(base) + step * rng.permutation(n).astype(np.float32) * 4)
        x = rng.normal(0, 1.5, n).astype(np.float32)
        x[rng.permutation(n)[:n // 2]] = np.float32(base) + step * rng.integers(0, 3, n // 2) * 2
        rows.append(x)
    x = np.stack(rows)
    for bias in (np.zeros(n), rng.integers(-2, 3, n) * 2.0 ** -12, rng.integers(0, 2, n) * 1e-7,
                 -2.0 + rng.integers(0, 3, n) * 2.0 ** -22, None):
        b = None if bias is None else bias.astype(np.float32).astype(np.float64)
        keep = groups_settled(x.astype(np.float64), b, *groups, score)
        assert keep.sum() >= len(x) // 2
        run(hip, x[keep], bias, k, *groups, score=score)


def groups_settled(x, bias, n_group, topk_group, group_top, score):
    """Rows whose kept groups 64-bit arithmetic settles. A group's count (s_a + b_1)
    + (s_b + b_2) and another's (s_a + b_2) + (s_b + b_1) are equal numbers, but
    each of the three additions may round by half of 2^-52 of a value below 4, so
    two such counts can come out up to 6 * 2^-52 * 4 / 2 < 2^-48 apart, in either
    order, by the last bits of s alone. Rows with counts that near at the border
    and not of the same logits and biases are left out."""
    keep = np.ones(len(x), bool)
    for t, l in enumerate(x):
        key = R.scores(l, score) + (0 if bias is None else bias)
        counts = []
        for g in np.arange(len(l)).reshape(n_group, -1):
            top = sorted(g, key=lambda e: (-key[e], e))[:group_top]
            counts.append((key[top].sum(), tuple(sorted((l[e], 0 if bias is None else bias[e]) for e in top))))
        counts.sort(key=lambda c: -c[0])
        if topk_group < n_group:
            edge = counts[topk_group - 1]
            keep[t] = all(c[1] == edge[1] or abs(c[0] - edge[0]) > 2.0 ** -48 for c in counts)
    return keep


@pytest.mark.parametrize("score", [0, 1, 2])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("groups", [(1, 1, 1), (8, 3, 2), (8, 3, 1)])
def test_masked_experts(hip, score, bias, groups):
    """-inf and NaN logits are never chosen, +inf ones first; rows with fewer
    experts than places, and with none."""
    rng = np.random.default_rng(7)
    x = rng.normal(0, 1.5, (12, 64))
    x[0] = -INF
    x[1] = NAN
    x[2, :] = -INF
    x[2, 40] = 1.0
    x[3, 1:] = -INF
    x[4, ::2] = NAN
    x[5, 8:] = -INF  # one group left
    x[6, 3] = x[6, 50] = INF if score != 2 else 1e30
    x[7, rng.permutation(64)[:59]] = -INF
    x[8] = np.where(rng.random(64) < 0.5, -INF, x[8])
    x[9] = -3.0e38
    x[10] = np.linspace(-800, -700, 64)
    b = rng.normal(0, 0.05, 64) if bias else None
    ids, w = run(hip, x, b, 6, *groups, score=score, scale=1.5)
    assert (ids[:2] == -1).all() and (w[:2] == 0).all()
    assert ids[2, 0] == 40 and (ids[2, 1:] == -1).all()


@pytest.mark.parametrize("groups", [(1, 1, 1), (4, 2, 2)])
def test_bias_switches_experts_off_and_on(hip, groups):
    rng = np.random.default_rng(8)
    x = rng.normal(0, 1.5, (9, 32))
    b = rng.normal(0, 0.05, 32)
    b[3], b[4], b[5], b[31] = -INF, NAN, INF, 100.0
    ids, _ = run(hip, x, b, 5, *groups, score=1)
    assert not np.isin(ids, (3, 4)).any()
    assert (ids[:, 0] == 5).all() and (ids[:, 1] == 31).all()
    run(hip, x, np.full(32, -INF), 5, *groups, score=0)
    run(hip, x, np.full(32, -7.5), 5, *groups, score=2)  # negative keys


def test_scale_and_renormalise(hip):
    rng = np.random.default_rng(9)
    x = rng.normal(0, 1.5, (6, 48))
    for score in (0, 1, 2):
        _, w = run(hip, x, None, 6, score=score, renorm=True, scale=1.0)
        np.testing.assert_allclose(w.sum(1), 1.0, rtol=6 * 2.0 ** -23)
        run(hip, x, None, 6, score=score, renorm=False, scale=-2.5)
        run(hip, x, None, 6, score=score, renorm=True, scale=0.0)


def test_many_tokens(hip):
    rng = np.random.default_rng(10)
    run(hip, rng.normal(0, 1.5, (2051, 256)), rng.normal(0, 0.05, 256), 8, 8, 4, 2, score=1)


def test_one_token_among_many_is_the_same_as_alone(hip):
    rng = np.random.default_rng(11)
    x = rng.normal(0, 1.5, (130, 256))
    b = rng.normal(0, 0.05, 256)
    ids, w = run(hip, x, b, 8, 8, 4, 2, score=1)
    for t in (0, 64, 129):
        i1, w1 = run(hip, x[t:t + 1], b, 8, 8, 4, 2, score=1)
        assert (i1 == ids[t]).all() and (w1 == w[t]).all()


def test_on_another_stream_and_captured(hip):
    rng = np.random.default_rng(12)
    s = torch.cuda.Stream()
    run(hip, rng.normal(0, 1.5, (9, 64)), None, 4, stream=s.cuda_stream)
    x = torch.zeros(9, 64, device="cuda")
    ids = torch.zeros(9, 4, dtype=torch.int32, device="cuda")
    w = torch.zeros(9, 4, device="cuda")

    def call(stream):
        hip.moe_route_dev(ids.data_ptr(), w.data_ptr(), 36, x.data_ptr(), 576, 64, 0, 0, 9, 64, 4,
                          score=2, scale=1.5, stream=stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(torch.cuda.current_stream().cuda_stream)
    for i in range(4):
        v = rng.normal(0, 1.5, (9, 64)).astype(np.float32)
        x.copy_(torch.from_numpy(v))
        g.replay()
        torch.cuda.synchronize()
        want_ids, want_w = R.route(v.astype(np.float64), None, 4, 1, 1, 1, 2, True, 1.5)
        np.testing.assert_array_equal(ids.cpu().numpy(), want_ids)
        np.testing.assert_allclose(w.cpu().numpy(), want_w, rtol=2.0 ** -23)
        ids.fill_(-5)


def test_rows_beyond_32_bit_offsets(hip):
    """4.6 GB of logits: the first and the last tokens."""
    n_tok, n, k = 4_500_001, 256, 8
    d = torch.randn(n_tok, n, device="cuda")
    b = torch.randn(n, device="cuda") * 0.05
    ids = torch.full((n_tok, k), -5, dtype=torch.int32, device="cuda")
    w = torch.zeros(n_tok, k, device="cuda")
    hip.moe_route_dev(ids.data_ptr(), w.data_ptr(), n_tok * k, d.data_ptr(), d.numel(), n, b.data_ptr(), n,
                      n_tok, n, k, 8, 4, 2, score=1, stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert (ids >= 0).all()
    for at in (slice(0, 9), slice(n_tok - 9, n_tok)):
        want_ids, want_w = R.route(d[at].cpu().double().numpy(), b.cpu().double().numpy(), k, 8, 4, 2, 1, True, 1.0)
        np.testing.assert_array_equal(ids[at].cpu().numpy(), want_ids)
        np.testing.assert_allclose(w[at].cpu().numpy(), want_w, rtol=2.0 ** -23)
