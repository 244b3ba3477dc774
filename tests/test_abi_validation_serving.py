"""Argument checks of the routing, int8-product and log-probability entry points.
Every refusal comes before any device work, so these run without a GPU; pointers
are made-up aligned addresses that are never read."""
import pytest

P = 1 << 40  # stands for a device pointer


def route(hip, **kw):
    a = dict(ids=P, weights=P, ids_len=4 * 2, logits=P, logits_len=4 * 16, stride=16, bias=0,
             bias_len=0, n_tok=4, n_expert=16, k=2, n_group=1, topk_group=1, group_top=1, score=0,
             renorm=True, scale=1.0, dtype=0)
    a.update(kw)
    hip.moe_route_dev(*a.values())


@pytest.mark.parametrize("kw,error,msg", [
    (dict(dtype=12), "Unimplemented", "dtype"),
    (dict(score=3), "InvalidArgument", "score"),
    (dict(n_expert=0), "InvalidArgument", "n_expert"),
    (dict(n_expert=16385, stride=16385, logits_len=4 * 16385), "InvalidArgument", "n_expert"),
    (dict(n_group=0), "InvalidArgument", "n_group"),
    (dict(n_group=3), "InvalidArgument", "n_group"),
    (dict(n_group=4, topk_group=0), "InvalidArgument", "topk_group"),
    (dict(n_group=4, topk_group=5), "InvalidArgument", "topk_group"),
    (dict(group_top=3), "InvalidArgument", "group_top"),
    (dict(k=0, ids_len=0), "InvalidArgument", "k must"),
    (dict(k=17, ids_len=68), "InvalidArgument", "k must"),
    (dict(n_group=4, topk_group=1, k=5, ids_len=20), "InvalidArgument", "k must"),
    (dict(n_expert=128, stride=128, logits_len=512, k=65, ids_len=260), "InvalidArgument", "k must"),
    (dict(scale=float("inf")), "InvalidArgument", "scale"),
    (dict(scale=float("nan")), "InvalidArgument", "scale"),
    (dict(stride=15), "ShapeMismatch", "logits"),
    (dict(logits_len=63), "ShapeMismatch", "logits"),
    (dict(stride=20, logits_len=75), "ShapeMismatch", "logits"),
    (dict(bias=P, bias_len=15), "ShapeMismatch", "bias"),
    (dict(ids_len=7), "ShapeMismatch", "ids"),
    (dict(n_tok=1 << 31, ids_len=1 << 32, logits_len=1 << 40), "ShapeMismatch", "n_tok"),
    (dict(logits=0), "InvalidArgument", "NULL"),
    (dict(ids=0), "InvalidArgument", "NULL"),
    (dict(weights=0), "InvalidArgument", "NULL"),
    (dict(bias=0, bias_len=16), "InvalidArgument", "NULL"),
    (dict(logits=P + 2), "InvalidArgument", "misaligned"),
    (dict(dtype=30, logits=P + 1), "InvalidArgument", "misaligned"),
    (dict(ids=P + 2), "InvalidArgument", "misaligned"),
])
def test_route_refusals(hip, kw, error, msg):
    with pytest.raises(getattr(hip, error), match=msg):
        route(hip, **kw)


def test_no_tokens_is_ok(hip):
    route(hip, n_tok=0, ids_len=0, logits_len=0, logits=0, ids=0, weights=0)
    quantize(hip, n_tok=0, x=0, x_len=0, xq=0, xq_len=0, scale=0, scale_len=0)
    prequant(hip, n_tok=0, out=0, out_len=0, xq=0, xq_len=0, xscale=0, xscale_len=0)
    oneshot(hip, n_tok=0, out=0, out_len=0, x=0, x_len=0)
    logprobs(hip, n_tok=0, out_len=0, top_len=0, logits=0, logits_len=0, tokens_len=0)


def quantize(hip, **kw):
    a = dict(x=P, x_len=3 * 100, stride=100, xq=P, xq_len=3 * 128, scale=P, scale_len=3, n_tok=3,
             in_dim=100, dtype=0)
    a.update(kw)
    hip.quantize_int8_dev(*a.values())


@pytest.mark.parametrize("kw,error,msg", [
    (dict(in_dim=0), "InvalidArgument", "in_dim"),
    (dict(in_dim=131072), "InvalidArgument", "in_dim"),
    (dict(dtype=8), "Unimplemented", "dtype"),
    (dict(stride=99), "ShapeMismatch", "x must"),
    (dict(x_len=299), "ShapeMismatch", "x must"),
    (dict(stride=110, x_len=319), "ShapeMismatch", "x must"),
    (dict(xq_len=300), "ShapeMismatch", "xq"),
    (dict(scale_len=2), "ShapeMismatch", "scale"),
    (dict(x=0), "InvalidArgument", "NULL"),
    (dict(xq=0), "InvalidArgument", "NULL"),
    (dict(scale=0), "InvalidArgument", "NULL"),
    (dict(x=P + 2), "InvalidArgument", "misaligned"),
    (dict(xq=P + 8), "InvalidArgument", "misaligned"),
])
def test_quantize_refusals(hip, kw, error, msg):
    with pytest.raises(getattr(hip, error), match=msg):
        quantize(hip, **kw)


def prequant(hip, **kw):
    a = dict(out=P, out_len=3 * 40, out_stride=40, w=P, w_len=40 * 128, ws=P, ws_len=40, bias=0,
             bias_len=0, xq=P, xq_len=3 * 128, xscale=P, xscale_len=3, work=P, work_len=None,
             n_tok=3, in_dim=100, out_dim=40, dtype_out=0)
    a.update(kw)
    if a["work_len"] is None:
        a["work_len"] = hip.int8_work_bytes(a["n_tok"], a["in_dim"], a["out_dim"])
    hip.matmul_int8_prequant_dev(*a.values())


def oneshot(hip, **kw):
    a = dict(out=P, out_len=3 * 40, out_stride=40, w=P, w_len=40 * 128, ws=P, ws_len=40, bias=0,
             bias_len=0, x=P, x_len=300, x_stride=100, work=P, work_len=None, n_tok=3, in_dim=100,
             out_dim=40, dtype_x=0, dtype_out=0)
    a.update(kw)
    if a["work_len"] is None:
        a["work_len"] = hip.int8_work_bytes(a["n_tok"], a["in_dim"], a["out_dim"])
    hip.matmul_int8_dev(*a.values())


PRODUCT = [
    (dict(dtype_out=8), "Unimplemented", "dtype"),
    (dict(in_dim=0), "InvalidArgument", "in_dim"),
    (dict(in_dim=131072), "InvalidArgument", "in_dim"),
    (dict(out_dim=0), "InvalidArgument", "out_dim"),
    (dict(w_len=40 * 100), "ShapeMismatch", "weights"),
    (dict(ws_len=39), "ShapeMismatch", "wscale"),
    (dict(bias=P, bias_len=3), "ShapeMismatch", "bias"),
    (dict(out_stride=39), "ShapeMismatch", "out must"),
    (dict(out_len=119), "ShapeMismatch", "out must"),
    (dict(out_stride=64, out_len=2 * 64 + 39), "ShapeMismatch", "out must"),
    (dict(w=0), "InvalidArgument", "NULL"),
    (dict(ws=0), "InvalidArgument", "NULL"),
    (dict(out=0), "InvalidArgument", "NULL"),
    (dict(bias=0, bias_len=40), "InvalidArgument", "NULL"),
    (dict(w=P + 8), "InvalidArgument", "misaligned"),
    (dict(out=P + 2), "InvalidArgument", "misaligned"),
    (dict(work=P + 16), "InvalidArgument", "misaligned"),
]


@pytest.mark.parametrize("kw,error,msg", PRODUCT + [
    (dict(xq_len=300), "ShapeMismatch", "xq"),
    (dict(xscale_len=4), "ShapeMismatch", "xscale"),
    (dict(xq=0), "InvalidArgument", "NULL"),
    (dict(xq=P + 4), "InvalidArgument", "misaligned"),
])
def test_prequant_refusals(hip, kw, error, msg):
    with pytest.raises(getattr(hip, error), match=msg):
        prequant(hip, **kw)


@pytest.mark.parametrize("kw,error,msg", PRODUCT + [
    (dict(dtype_x=8), "Unimplemented", "dtype"),
    (dict(x_stride=99), "ShapeMismatch", "x must"),
    (dict(x_len=299), "ShapeMismatch", "x must"),
    (dict(work_len=0), "ShapeMismatch", "work"),
    (dict(work=0), "InvalidArgument", "NULL"),
    (dict(x=0), "InvalidArgument", "NULL"),
])
def test_oneshot_refusals(hip, kw, error, msg):
    with pytest.raises(getattr(hip, error), match=msg):
        oneshot(hip, **kw)


def test_row_and_work_bytes(hip):
    assert [hip.int8_row_bytes(n) for n in (1, 64, 65, 4096, 131071)] == [64, 64, 128, 4096, 131072]
    assert hip.int8_row_bytes(0) == hip.int8_row_bytes(131072) == 0
    for t, k, n in ((1, 64, 64), (33, 100, 40), (300, 4096, 4096), (2048, 4096, 14336)):
        assert hip.int8_work_bytes(t, k, n) >= t * hip.int8_row_bytes(k) + 4 * t
    assert hip.int8_work_bytes(1, 0, 64) == hip.int8_work_bytes(1, 131072, 64) == 0
    assert hip.token_logprobs_work_bytes(1, 0, 0) == hip.token_logprobs_work_bytes(1, 100, 65) == 0


def logprobs(hip, **kw):
    a = dict(logprob=P, entropy=P, rank=P, out_len=3, top_ids=P, top=P, top_len=15, logits=P,
             logits_len=300, stride=100, tokens=P, tokens_len=3, work=P, work_len=None, n_tok=3,
             vocab=100, n_top=5, dtype=0)
    a.update(kw)
    if a["work_len"] is None:
        a["work_len"] = hip.token_logprobs_work_bytes(a["n_tok"], a["vocab"], a["n_top"])
    hip.token_logprobs_dev(*a.values())


@pytest.mark.parametrize("kw,error,msg", [
    (dict(dtype=8), "Unimplemented", "dtype"),
    (dict(vocab=0, n_top=0), "InvalidArgument", "vocab"),
    (dict(vocab=1 << 31, stride=1 << 31, logits_len=1 << 40), "InvalidArgument", "vocab"),
    (dict(n_top=65, top_len=195), "InvalidArgument", "n_top"),
    (dict(vocab=4, n_top=5), "InvalidArgument", "n_top"),
    (dict(stride=99), "ShapeMismatch", "logits"),
    (dict(logits_len=299), "ShapeMismatch", "logits"),
    (dict(tokens_len=2), "ShapeMismatch", "tokens"),
    (dict(out_len=4), "ShapeMismatch", "outputs"),
    (dict(top_len=14), "ShapeMismatch", "lists"),
    (dict(logits=0), "InvalidArgument", "NULL"),
    (dict(tokens=0), "InvalidArgument", "NULL"),
    (dict(logprob=0), "InvalidArgument", "NULL"),
    (dict(top_ids=0), "InvalidArgument", "NULL"),
    (dict(top=0), "InvalidArgument", "NULL"),
    (dict(logits=P + 2), "InvalidArgument", "misaligned"),
    (dict(dtype=1, logits=P + 1), "InvalidArgument", "misaligned"),
    (dict(rank=P + 1), "InvalidArgument", "misaligned"),
])
def test_logprobs_refusals(hip, kw, error, msg):
    with pytest.raises(getattr(hip, error), match=msg):
        logprobs(hip, **kw)


def test_logprobs_refuses_a_short_workspace(hip):
    """The largest workspace any size asks for, less one byte."""
    for n_tok, vocab in ((1, 200000), (7, 50000)):
        need = hip.token_logprobs_work_bytes(n_tok, vocab, 64)
        if need:
            with pytest.raises(hip.ShapeMismatch, match="work"):
                logprobs(hip, n_tok=n_tok, vocab=vocab, n_top=64, stride=vocab, top_len=64 * n_tok,
                         logits_len=n_tok * vocab, out_len=n_tok, tokens_len=n_tok,
                         work_len=need - 1)


LIMIT = (1 << 23) - 1  # rows and channels of one call: what every launch's grid can hold


def test_more_rows_or_channels_than_a_launch_holds(hip):
    n = LIMIT + 1
    with pytest.raises(hip.ShapeMismatch, match="8388607"):
        route(hip, n_tok=n, ids_len=2 * n, logits_len=16 * n)
    with pytest.raises(hip.ShapeMismatch, match="8388607"):
        quantize(hip, n_tok=n, x_len=1 << 40, xq_len=n * 128, scale_len=n)
    for call in (prequant, oneshot):
        for kw in (dict(n_tok=n), dict(out_dim=n, out_stride=n)):
            with pytest.raises(hip.ShapeMismatch, match="8388607"):
                call(hip, **kw)
    with pytest.raises(hip.ShapeMismatch, match="8388607"):
        logprobs(hip, n_tok=n, out_len=n, top_len=0, n_top=0, logits_len=1 << 40, tokens_len=n)
    assert hip.int8_work_bytes(n, 64, 64) == hip.int8_work_bytes(64, 64, n) == 0
    assert hip.int8_work_bytes(LIMIT, 64, LIMIT) > 0
    assert hip.token_logprobs_work_bytes(n, 64, 0) == 0
