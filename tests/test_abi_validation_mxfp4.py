"""Argument checks of the 4-bit floating-point entry points. Every refusal comes before
any device work, so these run without a GPU; pointers are made-up aligned addresses that
are never read."""
import pytest

from mxfp4_ref import row_bytes, scale_bytes

P = 1 << 40  # stands for a device pointer
K, RB, SB = 600, row_bytes(600), scale_bytes(600)


def test_sizes(hip):
    for n in (1, 2, 31, 128, 129, 512, 513, 4096, 1048576):
        assert hip.mxfp4_row_bytes(n) == row_bytes(n) and hip.mxfp4_scale_bytes(n) == scale_bytes(n)
    for n in (0, 1048577):
        assert hip.mxfp4_row_bytes(n) == 0 and hip.mxfp4_scale_bytes(n) == 0
        assert hip.mxfp4_work_bytes(4, n, 64) == 0
    assert hip.mxfp4_work_bytes(4, 64, 0) == 0 and hip.mxfp4_work_bytes(1 << 23, 64, 64) == 0
    assert hip.mxfp4_work_bytes(4, 64, 1 << 23) == 0
    sizes = [hip.mxfp4_work_bytes(t, 4096, 4096) for t in range(0, 600)]
    assert sizes == sorted(sizes)


def quantize(hip, **kw):
    a = dict(x=P, x_len=3 * K, stride=K, codes=P, codes_len=3 * RB, scales=P, scales_len=3 * SB, n_rows=3,
             in_dim=K, dtype=0)
    a.update(kw)
    hip.quantize_mxfp4_dev(*a.values())


def dequantize(hip, **kw):
    a = dict(codes=P, codes_len=3 * RB, scales=P, scales_len=3 * SB, x=P, x_len=3 * K, stride=K, n_rows=3,
             in_dim=K, dtype=0)
    a.update(kw)
    hip.dequantize_mxfp4_dev(*a.values())


@pytest.mark.parametrize("call", [quantize, dequantize])
@pytest.mark.parametrize("kw,error,msg", [
    (dict(in_dim=0), "InvalidArgument", "in_dim"),
    (dict(in_dim=1048577), "InvalidArgument", "in_dim"),
    (dict(n_rows=1 << 23), "ShapeMismatch", "n_rows"),
    (dict(dtype=8), "Unimplemented", "dtype"),
    (dict(stride=K - 1), "ShapeMismatch", "must hold"),
    (dict(x_len=3 * K - 1), "ShapeMismatch", "must hold"),
    (dict(stride=K + 5, x_len=3 * K + 9), "ShapeMismatch", "must hold"),
    (dict(codes_len=3 * RB - 1), "ShapeMismatch", "codes"),
    (dict(scales_len=3 * SB + 1), "ShapeMismatch", "scales"),
    (dict(x=0), "InvalidArgument", "NULL"),
    (dict(codes=0), "InvalidArgument", "NULL"),
    (dict(scales=0), "InvalidArgument", "NULL"),
    (dict(x=P + 2), "InvalidArgument", "misaligned"),
    (dict(x=P + 1, dtype=1), "InvalidArgument", "misaligned"),
    (dict(codes=P + 8), "InvalidArgument", "misaligned"),
    (dict(scales=P + 4), "InvalidArgument", "misaligned"),
])
def test_row_refusals(hip, call, kw, error, msg):
    with pytest.raises(getattr(hip, error), match=msg):
        call(hip, **kw)


def prequant(hip, **kw):
    a = dict(out=P, out_len=3 * 40, out_stride=40, w=P, w_len=40 * RB, ws=P, ws_len=40 * SB, bias=0, bias_len=0,
             xc=P, xc_len=3 * RB, xs=P, xs_len=3 * SB, work=P, work_len=None, n_tok=3, in_dim=K, out_dim=40,
             dtype_out=0)
    a.update(kw)
    if a["work_len"] is None:
        a["work_len"] = hip.mxfp4_work_bytes(a["n_tok"], a["in_dim"], a["out_dim"])
    hip.matmul_mxfp4_prequant_dev(*a.values())


def oneshot(hip, **kw):
    a = dict(out=P, out_len=3 * 40, out_stride=40, w=P, w_len=40 * RB, ws=P, ws_len=40 * SB, bias=0, bias_len=0,
             x=P, x_len=3 * K, x_stride=K, work=P, work_len=None, n_tok=3, in_dim=K, out_dim=40, dtype_x=0,
             dtype_out=0)
    a.update(kw)
    if a["work_len"] is None:
        a["work_len"] = hip.mxfp4_work_bytes(a["n_tok"], a["in_dim"], a["out_dim"])
    hip.matmul_mxfp4_dev(*a.values())


PRODUCT = [
    (dict(dtype_out=8), "Unimplemented", "dtype"),
    (dict(in_dim=0), "InvalidArgument", "in_dim"),
    (dict(in_dim=1048577), "InvalidArgument", "in_dim"),
    (dict(out_dim=0), "InvalidArgument", "out_dim"),
    (dict(out_dim=1 << 23), "ShapeMismatch", "out_dim"),
    (dict(n_tok=1 << 23), "ShapeMismatch", "n_tok"),
    (dict(w_len=40 * RB - 64), "ShapeMismatch", "weights"),
    (dict(ws_len=39 * SB), "ShapeMismatch", "weights"),
    (dict(bias=P, bias_len=3), "ShapeMismatch", "bias"),
    (dict(out_stride=39), "ShapeMismatch", "out must"),
    (dict(out_len=119), "ShapeMismatch", "out must"),
    (dict(out_stride=64, out_len=2 * 64 + 39), "ShapeMismatch", "out must"),
    (dict(work_len=255), "ShapeMismatch", "work"),
    (dict(w=0), "InvalidArgument", "NULL"),
    (dict(ws=0), "InvalidArgument", "NULL"),
    (dict(out=0), "InvalidArgument", "NULL"),
    (dict(work=0), "InvalidArgument", "NULL"),
    (dict(bias=0, bias_len=40), "InvalidArgument", "NULL"),
    (dict(w=P + 8), "InvalidArgument", "misaligned"),
    (dict(ws=P + 8), "InvalidArgument", "misaligned"),
    (dict(out=P + 2), "InvalidArgument", "misaligned"),
    (dict(bias=P + 2, bias_len=40), "InvalidArgument", "misaligned"),
    (dict(work=P + 16), "InvalidArgument", "misaligned"),
]


@pytest.mark.parametrize("kw,error,msg", PRODUCT + [
    (dict(xc_len=2 * RB), "ShapeMismatch", "xcodes"),
    (dict(xs_len=4 * SB), "ShapeMismatch", "xcodes"),
    (dict(xc=0), "InvalidArgument", "NULL"),
    (dict(xs=0), "InvalidArgument", "NULL"),
    (dict(xc=P + 4), "InvalidArgument", "misaligned"),
])
def test_prequant_refusals(hip, kw, error, msg):
    with pytest.raises(getattr(hip, error), match=msg):
        prequant(hip, **kw)


@pytest.mark.parametrize("kw,error,msg", PRODUCT + [
    (dict(dtype_x=8), "Unimplemented", "dtype"),
    (dict(x_stride=K - 1), "ShapeMismatch", "x must"),
    (dict(x_len=3 * K - 1), "ShapeMismatch", "x must"),
    (dict(x=0), "InvalidArgument", "NULL"),
    (dict(x=P + 2), "InvalidArgument", "misaligned"),
])
def test_product_refusals(hip, kw, error, msg):
    with pytest.raises(getattr(hip, error), match=msg):
        oneshot(hip, **kw)


E, D, F, SH = 8, 300, 200, 1


def layer(hip, **kw):
    rows, down = (E + SH) * F, (E + SH) * D
    a = dict(router=P, router_len=E * D, dtype_router=0, bias=0, bias_len=0, gate=P, up=P,
             gate_up_len=rows * row_bytes(D), gate_scales=P, up_scales=P, gate_up_scales_len=rows * scale_bytes(D),
             down=P, down_len=down * row_bytes(F), down_scales=P, down_scales_len=down * scale_bytes(F), n_embd=D,
             n_ff=F, n_expert=E, n_shared=SH, k=2, n_group=1, topk_group=1, group_top=1, score=0, renormalise=1,
             scale=1.0, clamp=0.0)
    a.update(kw)
    return hip.MoeMxfp4(**a)


def moe(hip, lay=None, **kw):
    lay = lay or layer(hip)
    a = dict(out=P, out_len=3 * D, out_stride=D, ids=P, weights=P, ids_len=6, x=P, x_len=3 * D, x_stride=D, work=P,
             work_len=hip.moe_mxfp4_work_bytes(lay, 3), n_tok=3, dtype_x=0, dtype_out=0)
    a.update(kw)
    hip.moe_mxfp4_dev(lay, *a.values())


@pytest.mark.parametrize("kw,error,msg", [
    (dict(dtype_router=8), "Unimplemented", "router"),
    (dict(score=3), "InvalidArgument", "score"),
    (dict(n_embd=0), "InvalidArgument", "n_embd"),
    (dict(n_embd=65537), "InvalidArgument", "n_embd"),
    (dict(n_ff=0), "InvalidArgument", "n_ff"),
    (dict(n_ff=65537), "InvalidArgument", "n_ff"),
    (dict(n_expert=0), "InvalidArgument", "n_expert"),
    (dict(n_expert=1025), "InvalidArgument", "n_expert"),
    (dict(n_shared=9), "InvalidArgument", "n_shared"),
    (dict(k=0), "InvalidArgument", "k"),
    (dict(k=33), "InvalidArgument", "k"),
    (dict(k=9), "InvalidArgument", "k"),
    (dict(n_group=4, topk_group=1, k=3), "InvalidArgument", "k"),
    (dict(n_group=0), "InvalidArgument", "n_group"),
    (dict(n_group=3), "InvalidArgument", "n_group"),
    (dict(n_group=4, topk_group=0), "InvalidArgument", "topk_group"),
    (dict(n_group=4, topk_group=5), "InvalidArgument", "topk_group"),
    (dict(group_top=3), "InvalidArgument", "group_top"),
    (dict(scale=float("inf")), "InvalidArgument", "scale"),
    (dict(clamp=float("nan")), "InvalidArgument", "clamp"),
    (dict(router_len=E * D - 1), "ShapeMismatch", "router"),
    (dict(bias=P, bias_len=7), "ShapeMismatch", "bias"),
    (dict(gate_up_len=1), "ShapeMismatch", "gate"),
    (dict(gate_up_scales_len=1), "ShapeMismatch", "gate"),
    (dict(n_shared=2), "ShapeMismatch", "gate"),
    (dict(down_len=1), "ShapeMismatch", "down"),
    (dict(down_scales_len=1), "ShapeMismatch", "down"),
    (dict(router=0), "InvalidArgument", "NULL"),
    (dict(bias_len=8), "InvalidArgument", "NULL"),
    (dict(gate=0), "InvalidArgument", "NULL"),
    (dict(up=0), "InvalidArgument", "NULL"),
    (dict(up_scales=0), "InvalidArgument", "NULL"),
    (dict(down=0), "InvalidArgument", "NULL"),
    (dict(router=P + 2), "InvalidArgument", "misaligned"),
    (dict(bias=P + 2, bias_len=8), "InvalidArgument", "misaligned"),
    (dict(gate=P + 8), "InvalidArgument", "misaligned"),
    (dict(up_scales=P + 8), "InvalidArgument", "misaligned"),
    (dict(down_scales=P + 1), "InvalidArgument", "misaligned"),
])
def test_layer_refusals(hip, kw, error, msg):
    with pytest.raises(getattr(hip, error), match=msg):
        moe(hip, layer(hip, **kw), work_len=1 << 40)


@pytest.mark.parametrize("kw,error,msg", [
    (dict(n_tok=33, work_len=1 << 40), "InvalidArgument", "n_tok"),
    (dict(dtype_x=8), "Unimplemented", "dtype"),
    (dict(dtype_out=12), "Unimplemented", "dtype"),
    (dict(out_stride=D - 1), "ShapeMismatch", "out must"),
    (dict(out_len=3 * D - 1), "ShapeMismatch", "out must"),
    (dict(x_stride=D - 1), "ShapeMismatch", "x must"),
    (dict(x_stride=D + 4, x_len=3 * D + 7), "ShapeMismatch", "x must"),
    (dict(ids_len=5), "ShapeMismatch", "ids"),
    (dict(work_len=100), "ShapeMismatch", "work"),
    (dict(out=0), "InvalidArgument", "NULL"),
    (dict(x=0), "InvalidArgument", "NULL"),
    (dict(ids=0), "InvalidArgument", "NULL"),
    (dict(weights=0), "InvalidArgument", "NULL"),
    (dict(work=0), "InvalidArgument", "NULL"),
    (dict(x=P + 2), "InvalidArgument", "misaligned"),
    (dict(out=P + 1, dtype_out=30), "InvalidArgument", "misaligned"),
    (dict(ids=P + 2), "InvalidArgument", "misaligned"),
    (dict(work=P + 128), "InvalidArgument", "misaligned"),
])
def test_moe_refusals(hip, kw, error, msg):
    with pytest.raises(getattr(hip, error), match=msg):
        moe(hip, **kw)


def test_no_layer(hip):
    import ctypes
    assert hip.LIB.rsllm_hip_moe_mxfp4_work_bytes(None, 3) == 0
    assert hip.LIB.rsllm_hip_moe_mxfp4_dev(None, P, D, D, P, P, 2, P, D, D, P, 1 << 30, 1, 0, 0,
                                           ctypes.c_void_p(None)) == hip.ERR_INVALID_ARGUMENT


def test_moe_work_bytes(hip):
    sizes = [hip.moe_mxfp4_work_bytes(layer(hip), t) for t in range(33)]
    assert sizes == sorted(sizes) and sizes[1] > 0
    assert hip.moe_mxfp4_work_bytes(layer(hip), 33) == 0
    assert hip.moe_mxfp4_work_bytes(layer(hip, n_expert=1025), 3) == 0


def test_no_tokens_is_ok(hip):
    quantize(hip, n_rows=0, x=0, x_len=0, codes=0, codes_len=0, scales=0, scales_len=0)
    dequantize(hip, n_rows=0, x=0, x_len=0, codes=0, codes_len=0, scales=0, scales_len=0)
    prequant(hip, n_tok=0, out=0, out_len=0, xc=0, xc_len=0, xs=0, xs_len=0, work=0, work_len=0)
    oneshot(hip, n_tok=0, out=0, out_len=0, x=0, x_len=0, work=0, work_len=0)
    moe(hip, n_tok=0, out=0, out_len=0, ids=0, weights=0, ids_len=0, x=0, x_len=0, work=0,
        work_len=hip.moe_mxfp4_work_bytes(layer(hip), 0))
