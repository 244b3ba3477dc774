"""The microscaled 4-bit calls that this backend is timed on (quantising, the product,
a whole mixture-of-experts layer), beside a plain form of each in torch operations.

Kinds
  roundtrip quantize_mxfp4_dev, then dequantize_mxfp4_dev: the values that 4-bit codes
            with a scale for every 32 of them stand for
  matmul    matmul_mxfp4_dev: float activations, quantised on the way, through one matrix
  pair      quantize_mxfp4_dev once, then matmul_mxfp4_prequant_dev on two matrices
            (an FFN's gate and up projections)
  moe       moe_mxfp4_dev: a few tokens through a router, the experts it chooses and
            those that every token takes, whose weights are 4-bit

Values: activations N(0, 1) with a few large channels, weights the codes of normal rows,
router weights of such a size that its logits are N(0, 1.5), balancing biases N(0, 0.05).
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GGML = {"f32": 0, "f16": 1, "bf16": 30}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
SCORES = {"softmax": 0, "sigmoid": 1, "sqrt_softplus": 2}
GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
# no drawn case does more than the largest listed one of its kind
MAX_ELEMENTS = 14336 * 4096
MAX_OPS = 2 * 2048 * 4096 * 14336
MAX_PAIRS = 32 * 7 * 4096 * 2048
MAX_EXPERTS = 257 * 4096 * 2048


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # One decoded token's activations as the 4-bit path sees them: all latency.
        {"name": "roundtrip_t1", "kind": "roundtrip", "tok": 1, "in": 4096, "x": "f32", "y": "f32", "pad": 0},
        # A dense FFN matrix converted when a model is loaded.
        {"name": "roundtrip_weight", "kind": "roundtrip", "tok": 14336, "in": 4096, "x": "bf16", "y": "bf16", "pad": 0},
        # A dense FFN's up projection, one decoded token: the weight stream.
        {"name": "matmul_t1", "kind": "matmul", "in": 4096, "out": 14336, "tok": 1, "x": "f32",
         "y": "f32", "bias": False, "pad": 0},
        # A projection with a bias for a full decode batch.
        {"name": "matmul_t32", "kind": "matmul", "in": 4096, "out": 4096, "tok": 32, "x": "bf16",
         "y": "bf16", "bias": True, "pad": 0},
        # Sizes that no tile divides, rows further apart than they are long.
        {"name": "matmul_odd", "kind": "matmul", "in": 2000, "out": 1001, "tok": 77, "x": "f16",
         "y": "f32", "bias": True, "pad": 24},
        # Gate and up over a prompt of ragged length, quantised once.
        {"name": "pair_t300", "kind": "pair", "in": 4096, "out": 2048, "tok": 300,
         "x": "f32", "y": "f32", "bias": False, "pad": 0},
        # A dense FFN's up projection over a long prompt: the matrix cores.
        {"name": "matmul_t2048", "kind": "matmul", "in": 4096, "out": 14336, "tok": 2048, "x": "bf16",
         "y": "bf16", "bias": False, "pad": 0},
        # A small layer of odd sizes with grouped experts: latency.
        {"name": "moe_odd_t5", "kind": "moe", "embd": 1000, "ff": 352, "experts": 32, "shared": 0, "top": 4,
         "groups": 4, "top_groups": 2, "group_top": 2, "score": "sigmoid", "route_bias": True, "renorm": True,
         "scale": 2.5, "clamp": 0.0, "tok": 5, "x": "f16", "y": "f16", "router": "f32", "pad": 8},
        # One decoded token through DS-V4's layer: 6 of 256 experts and the shared one.
        {"name": "moe_dsv4_t1", "kind": "moe", "embd": 4096, "ff": 2048, "experts": 256, "shared": 1, "top": 6,
         "groups": 1, "top_groups": 1, "group_top": 1, "score": "sqrt_softplus", "route_bias": True, "renorm": True,
         "scale": 1.5, "clamp": 10.0, "tok": 1, "x": "f32", "y": "f32", "router": "f32", "pad": 0},
        # A small decode batch over few wide experts, 8 of 64.
        {"name": "moe_e64_t8", "kind": "moe", "embd": 7168, "ff": 2048, "experts": 64, "shared": 0, "top": 8,
         "groups": 1, "top_groups": 1, "group_top": 1, "score": "softmax", "route_bias": False, "renorm": True,
         "scale": 1.0, "clamp": 0.0, "tok": 8, "x": "bf16", "y": "bf16", "router": "bf16", "pad": 0},
        # A full decode batch through DS-V4's layer: more than half of its experts.
        {"name": "moe_dsv4_t32", "kind": "moe", "embd": 4096, "ff": 2048, "experts": 256, "shared": 1, "top": 6,
         "groups": 1, "top_groups": 1, "group_top": 1, "score": "sqrt_softplus", "route_bias": True, "renorm": True,
         "scale": 1.5, "clamp": 10.0, "tok": 32, "x": "f32", "y": "f32", "router": "f32", "pad": 0},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choices(["roundtrip", "matmul", "pair", "moe"], [3, 6, 2, 6])[0]
    case = {"kind": kind, "x": rng.choice(["f32", "bf16", "f16"]), "y": rng.choice(["f32", "bf16", "f16"]),
            "pad": rng.choice([0, 0, 3, 64])}
    if kind == "roundtrip":
        in_dim = _log_int(rng, 32, 16384)
        return {**case, "in": in_dim, "tok": _log_int(rng, 1, MAX_ELEMENTS // in_dim)}
    if kind == "moe":
        groups = rng.choice([1, 1, 1, 4, 8])
        experts = groups * _log_int(rng, max(4, 8 // groups), 256 // groups)
        top_groups = rng.randint(1, groups)
        # whole blocks mostly, odd sizes now and then
        whole = rng.random() < 0.75
        embd = 32 * _log_int(rng, 8, 224) if whole else _log_int(rng, 200, 7168)
        ff = 32 * _log_int(rng, 4, 128) if whole else _log_int(rng, 100, 4096)
        top = min(_log_int(rng, 1, 10), experts // groups * top_groups)
        shared = rng.choice([0, 0, 1, 2])
        while (experts + shared) * embd * ff > MAX_EXPERTS:
            ff = (ff + 1) // 2
        tok = max(1, min(_log_int(rng, 1, 32), MAX_PAIRS // ((top + shared) * embd * ff)))
        return {**case, "embd": embd, "ff": ff, "experts": experts, "shared": shared, "top": top, "groups": groups,
                "top_groups": top_groups, "group_top": rng.choice([1, 2]), "score": rng.choice(sorted(SCORES)),
                "route_bias": rng.random() < 0.6, "renorm": rng.random() < 0.7, "scale": rng.choice([1.0, 1.5, 2.5]),
                "clamp": rng.choice([0.0, 7.0, 10.0]), "tok": tok, "router": rng.choice(["f32", "bf16", "f16"])}
    in_dim = 32 * _log_int(rng, 8, 448) if rng.random() < 0.75 else _log_int(rng, 200, 14000)
    out = 64 * _log_int(rng, 2, 256) if rng.random() < 0.75 else _log_int(rng, 100, 16000)
    tok = _log_int(rng, 1, 32) if rng.random() < 0.5 else _log_int(rng, 33, 2048)
    mats = 2 if kind == "pair" else 1
    return {**case, "in": in_dim, "out": out, "tok": max(1, min(tok, MAX_OPS // (2 * mats * in_dim * out))),
            "bias": rng.random() < 0.3}


def _row(n):
    """Bytes of a row of n codes: two a byte, whole 64-byte pieces."""
    return (n + 127) // 128 * 64


def _scale_row(n):
    """Bytes of a row's scales: one for 32 codes, whole 16-byte pieces."""
    return (n + 511) // 512 * 16


# ---------------------------------------------------------------------------
# Inputs, on the GPU, from the seed alone
# ---------------------------------------------------------------------------

def _gen(seed, stream):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + stream * 7919) % (1 << 62))
    return g


def _randn(shape, seed, stream):
    return torch.randn(*shape, device="cuda", generator=_gen(seed, stream))


def _empty(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device="cuda")


def _strided(values, pad):
    """The same values in rows that lie `pad` elements further apart."""
    if not pad:
        return values.contiguous()
    base = torch.zeros(values.shape[0], values.shape[1] + pad, dtype=values.dtype, device="cuda")
    base[:, :values.shape[1]] = values
    return base[:, :values.shape[1]]


def _weights(rows, in_dim, seed, stream):
    """A 4-bit matrix as a program keeps it: codes as often as the values of normal rows
    have them, and scales near those of rows of length 1. Codes and scales behind a
    row's end are 0."""
    # 256 pairs of codes, of normal values over a block's scale (its largest of 32 near 5)
    g = torch.Generator()
    g.manual_seed(5)
    v = torch.randn(256, 2, generator=g) * 2.0
    grid = torch.tensor(GRID)
    near = (v.abs()[:, :, None] - grid).abs().argmin(2)
    table = (near + 8 * (v < 0)).to(torch.uint8)
    table = (table[:, 0] + 16 * table[:, 1]).cuda()
    codes = torch.zeros(rows, _row(in_dim), dtype=torch.uint8, device="cuda")
    gen = _gen(seed, stream)
    step = max(1, (1 << 28) // codes.shape[1])
    for r in range(0, rows, step):
        pick = torch.randint(0, 256, (min(step, rows - r), (in_dim + 1) // 2), device="cuda", generator=gen,
                             dtype=torch.uint8)
        codes[r:r + step, :(in_dim + 1) // 2] = table[pick.int()]
    if in_dim % 2:
        codes[:, in_dim // 2] &= 15
    scales = torch.zeros(rows, _scale_row(in_dim), dtype=torch.uint8, device="cuda")
    blocks = (in_dim + 31) // 32
    at = 127 + int(round(math.log2(0.5 / math.sqrt(in_dim))))
    scales[:, :blocks] = torch.randint(at - 1, at + 2, (rows, blocks), device="cuda", generator=gen,
                                       dtype=torch.uint8)
    return codes, scales


def _activations(tok, in_dim, dtype, pad, seed):
    x = _randn((tok, in_dim), seed, 1)
    x *= 1.0 + 15.0 * (torch.rand(in_dim, device="cuda", generator=_gen(seed, 2)) < 0.005)
    return _strided(x.to(DTYPES[dtype]), pad)


def prepare(case, seed):
    kind, t = case["kind"], case["tok"]
    s = {"case": case, "stream": torch.cuda.current_stream().cuda_stream}
    if kind == "moe":
        d, f, n = case["embd"], case["ff"], case["experts"]
        s["x"] = _activations(t, d, case["x"], case["pad"], seed)
        s["router"] = (_randn((n, d), seed, 3) * (1.5 / math.sqrt(d))).to(DTYPES[case["router"]])
        s["bias"] = _randn((n,), seed, 4) * 0.05 if case["route_bias"] else None
        stacked = n + case["shared"]
        s["gate"] = _weights(stacked * f, d, seed, 5)
        s["up"] = _weights(stacked * f, d, seed, 6)
        s["down"] = _weights(stacked * d, f, seed, 7)
        s["out"] = _empty(t, d, dtype=DTYPES[case["y"]])
        s["ids"], s["weights"] = _empty(t, case["top"], dtype=torch.int32), _empty(t, case["top"])
        return s
    k = case["in"]
    s["x"] = _activations(t, k, case["x"], case["pad"], seed)
    s["xcodes"] = _empty(t, _row(k), dtype=torch.uint8)
    s["xscales"] = _empty(t, _scale_row(k), dtype=torch.uint8)
    if kind == "roundtrip":
        s["y"] = _empty(t, k, dtype=DTYPES[case["y"]])
        return s
    n = case["out"]
    s["w"] = [_weights(n, k, seed, 10 + i) for i in range(2 if kind == "pair" else 1)]
    s["bias"] = _randn((n,), seed, 3) if case["bias"] else None
    s["y"] = [_empty(t, n, dtype=DTYPES[case["y"]]) for _ in s["w"]]
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def _work(s, B, name, *dims):
    """The call's workspace, which a program keeps from one call to the next."""
    if "work" not in s:
        s["work"] = _empty(max(1, getattr(B, name)(*dims)), dtype=torch.uint8)
    return s["work"].data_ptr(), s["work"].numel()


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _span(t):
    """Elements from a matrix's first to its last."""
    return (t.shape[0] - 1) * t.stride(0) + t.shape[1]


def _quantize_own(s, B, c):
    x, xc, xs = s["x"], s["xcodes"], s["xscales"]
    B.quantize_mxfp4_dev(x.data_ptr(), _span(x), x.stride(0), xc.data_ptr(), xc.numel(), xs.data_ptr(),
                         xs.numel(), c["tok"], c["in"], GGML[c["x"]], s["stream"])


def _roundtrip_own(s, c):
    from rsllm_amd import backend as B
    _quantize_own(s, B, c)
    xc, xs, y = s["xcodes"], s["xscales"], s["y"]
    B.dequantize_mxfp4_dev(xc.data_ptr(), xc.numel(), xs.data_ptr(), xs.numel(), y.data_ptr(), y.numel(),
                           y.stride(0), c["tok"], c["in"], GGML[c["y"]], s["stream"])
    return {"values": y}


def _matmul_own(s, c):
    from rsllm_amd import backend as B
    x, t, k, n = s["x"], c["tok"], c["in"], c["out"]
    work, work_len = _work(s, B, "mxfp4_work_bytes", t, k, n)
    nb = n if c["bias"] else 0
    if c["kind"] == "matmul":
        (w, ws), y = s["w"][0], s["y"][0]
        B.matmul_mxfp4_dev(y.data_ptr(), t * n, n, w.data_ptr(), w.numel(), ws.data_ptr(), ws.numel(),
                           _ptr(s["bias"]), nb, x.data_ptr(), _span(x), x.stride(0), work, work_len,
                           t, k, n, GGML[c["x"]], GGML[c["y"]], s["stream"])
        return {"y0": y}
    _quantize_own(s, B, c)
    xc, xs = s["xcodes"], s["xscales"]
    for (w, ws), y in zip(s["w"], s["y"]):
        B.matmul_mxfp4_prequant_dev(y.data_ptr(), t * n, n, w.data_ptr(), w.numel(), ws.data_ptr(), ws.numel(),
                                    _ptr(s["bias"]), nb, xc.data_ptr(), xc.numel(), xs.data_ptr(), xs.numel(),
                                    work, work_len, t, k, n, GGML[c["y"]], s["stream"])
    return {"y0": s["y"][0], "y1": s["y"][1]}


def _moe_own(s, c):
    from rsllm_amd import backend as B
    if "layer" not in s:  # which a program makes once
        r, (g, gs), (u, us), (w, ws) = s["router"], s["gate"], s["up"], s["down"]
        s["layer"] = B.MoeMxfp4(
            router=r.data_ptr(), router_len=r.numel(), dtype_router=GGML[c["router"]], bias=_ptr(s["bias"]),
            bias_len=c["experts"] if c["route_bias"] else 0, gate=g.data_ptr(), up=u.data_ptr(), gate_up_len=g.numel(),
            gate_scales=gs.data_ptr(), up_scales=us.data_ptr(), gate_up_scales_len=gs.numel(), down=w.data_ptr(),
            down_len=w.numel(), down_scales=ws.data_ptr(), down_scales_len=ws.numel(), n_embd=c["embd"],
            n_ff=c["ff"], n_expert=c["experts"], n_shared=c["shared"], k=c["top"], n_group=c["groups"],
            topk_group=c["top_groups"], group_top=c["group_top"], score=SCORES[c["score"]],
            renormalise=int(c["renorm"]), scale=c["scale"], clamp=c["clamp"])
    x, out, t = s["x"], s["out"], c["tok"]
    work, work_len = _work(s, B, "moe_mxfp4_work_bytes", s["layer"], t)
    B.moe_mxfp4_dev(s["layer"], out.data_ptr(), out.numel(), out.stride(0), s["ids"].data_ptr(),
                    s["weights"].data_ptr(), s["ids"].numel(), x.data_ptr(), _span(x), x.stride(0), work, work_len,
                    t, GGML[c["x"]], GGML[c["y"]], s["stream"])
    return {"out": out, "ids": s["ids"], "weights": s["weights"]}


def _quantised(x):
    """x (float) as the values its 4-bit codes stand for, in 64 bits."""
    t, k = x.shape
    blocks = (k + 31) // 32
    v = torch.zeros(t, blocks * 32, dtype=torch.float64, device=x.device)
    v[:, :k] = x
    v = v.view(t, blocks, 32)
    top = v.abs().amax(2, keepdim=True)
    e = torch.where(top > 0, torch.frexp(top).exponent - 3, torch.full_like(top, -127, dtype=torch.int32))
    unit = torch.exp2(e.clamp(-127, 127).double())
    v = v / unit
    step = torch.exp2((torch.frexp(v).exponent - 2).clamp(-1, 1).double())
    v = ((v / step).round() * step).clamp(-6.0, 6.0) * unit
    return v.view(t, blocks * 32)[:, :k]


def _values(codes, scales, in_dim):
    """Rows of codes and scales as the f32 values they stand for."""
    grid = torch.tensor(GRID + [-g for g in GRID], device=codes.device)
    v = torch.stack([grid[(codes & 15).int()], grid[(codes >> 4).int()]], 2).view(codes.shape[0], -1)
    blocks = (in_dim + 31) // 32
    unit = torch.exp2(scales[:, :blocks].double() - 127.0).float()
    return (v[:, :blocks * 32].reshape(-1, blocks, 32) * unit[:, :, None]).view(-1, blocks * 32)[:, :in_dim]


def _roundtrip_plain(s, c):
    # which code is nearest is decided in 64 bits
    x = s["x"]
    step = max(1, (1 << 24) // c["in"])
    y = [_quantised(x[r:r + step].double()).to(DTYPES[c["y"]]) for r in range(0, c["tok"], step)]
    return {"values": torch.cat(y)}


def _matmul_plain(s, c):
    q = _quantised(s["x"].double()).float()
    out = {}
    for i, (w, ws) in enumerate(s["w"]):
        y = q @ _values(w, ws, c["in"]).t()
        if s["bias"] is not None:
            y = y + s["bias"]
        out["y%d" % i] = y.to(DTYPES[c["y"]])
    return out


def _route_plain(s, c):
    # logits and scores in 64 bits: the ids go by which of two near ones is larger
    x = s["x"].double() @ s["router"].double().t()
    if c["score"] == "softmax":
        e = torch.exp(x - x.amax(1, keepdim=True))
        score = e / e.sum(1, keepdim=True)
    elif c["score"] == "sigmoid":
        score = 1.0 / (1.0 + torch.exp(-x))
    else:
        score = torch.sqrt(x.clamp(min=0) + torch.log1p(torch.exp(-x.abs())))
    key = score if s["bias"] is None else score + s["bias"].double()
    t, n = key.shape
    if c["groups"] > 1:
        inside = key.view(t, c["groups"], n // c["groups"])
        best = inside.sort(dim=2, descending=True).values[:, :, :c["group_top"]].sum(2)
        order = best.sort(dim=1, descending=True, stable=True).indices[:, :c["top_groups"]]
        kept = torch.zeros_like(best, dtype=torch.bool).scatter_(1, order, True)
        key = inside.masked_fill(~kept[:, :, None], -math.inf).view(t, n)
    ids = key.sort(dim=1, descending=True, stable=True).indices[:, :c["top"]]
    w = score.gather(1, ids)
    if c["renorm"]:
        w = w / w.sum(1, keepdim=True)
    return ids, (w * c["scale"]).float()


def _swiglu(g, u, clamp):
    if clamp > 1e-6:
        g, u = g.clamp(max=clamp), u.clamp(-clamp, clamp)
    return g / (1.0 + torch.exp(-g)) * u


def _moe_plain(s, c):
    ids, weights = _route_plain(s, c)
    x, d, f = s["x"].float(), c["embd"], c["ff"]
    out = torch.zeros(c["tok"], d, device=x.device)
    experts = torch.unique(ids).tolist() + list(range(c["experts"], c["experts"] + c["shared"]))
    for e in experts:
        if e < c["experts"]:
            tok, slot = (ids == e).nonzero(as_tuple=True)
            w = weights[tok, slot][:, None]
        else:
            tok, w = torch.arange(c["tok"], device=x.device), 1.0
        mine = x[tok]
        g, u = (mine @ _values(m[0][e * f:(e + 1) * f], m[1][e * f:(e + 1) * f], d).t() for m in (s["gate"], s["up"]))
        down = _values(s["down"][0][e * d:(e + 1) * d], s["down"][1][e * d:(e + 1) * d], f)
        out[tok] += (_swiglu(g, u, c["clamp"]) @ down.t()) * w
    return {"out": out.to(DTYPES[c["y"]]), "ids": ids.to(torch.int32), "weights": weights}


def run(s):
    c = s["case"]
    if own:
        return {"roundtrip": _roundtrip_own, "moe": _moe_own}.get(c["kind"], _matmul_own)(s, c)
    return {"roundtrip": _roundtrip_plain, "moe": _moe_plain}.get(c["kind"], _matmul_plain)(s, c)


# ---------------------------------------------------------------------------
# What a pass cannot do without, and its results in 64 bits
# ---------------------------------------------------------------------------

def _held(rows, in_dim):
    """Bytes of a matrix of codes and scales."""
    return rows * (in_dim + 1) // 2 + rows * ((in_dim + 31) // 32)


def work(case):
    t, x, y = case["tok"], SIZE[case["x"]], SIZE[case["y"]]
    if case["kind"] == "moe":
        d, f, n, k = case["embd"], case["ff"], case["experts"], case["top"]
        # how many experts the tokens are likely to choose between them
        chosen = n * (1.0 - (1.0 - k / n) ** t) + case["shared"]
        return {"bytes": int(chosen * (2 * _held(f, d) + _held(d, f))) + n * d * SIZE[case["router"]]
                + t * d * (x + y) + t * k * 8,
                "flops": t * (k + case["shared"]) * 6 * d * f + 2 * t * n * d}
    k = case["in"]
    if case["kind"] == "roundtrip":
        return {"bytes": t * k * (x + y) + 2 * _held(t, k), "flops": t * k * 4}
    n, mats = case["out"], 2 if case["kind"] == "pair" else 1
    return {"bytes": t * k * x + mats * (_held(n, k) + t * n * y) + (4 * n if case["bias"] else 0),
            "flops": 2 * mats * t * k * n}


def _decode_exact(codes, scales, in_dim):
    """(codes, scales) of rows in 64 bits, bit field by bit field."""
    both = torch.empty(codes.shape[0], 2 * codes.shape[1], dtype=torch.float64, device=codes.device)
    for half in range(2):
        c = (codes >> (4 * half)).int() & 15
        power, frac = (c >> 1) & 3, (c & 1).double()
        size = torch.where(power == 0, 0.5 * frac, torch.ldexp(1.0 + 0.5 * frac, power - 1))
        both[:, half::2] = torch.where(c >= 8, -size, size)
    unit = torch.ldexp(torch.ones((), dtype=torch.float64, device=codes.device), scales.int() - 127)
    return both[:, :in_dim] * unit.repeat_interleave(32, 1)[:, :in_dim]


def _nearest_exact(x):
    """Rows of x as their 4-bit values, by looking for the nearest of all codes."""
    t, k = x.shape
    out = torch.zeros(t, k, dtype=torch.float64, device=x.device)
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64, device=x.device)
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    for b in range(0, k, 32):
        v = x[:, b:b + 32].double()
        top = v.abs().amax(1)
        e = torch.where(top > 0, torch.floor(torch.log2(top)), -125.0)
        # where the logarithm rounded
        e = e + (top >= torch.exp2(e + 1)).double() - ((top < torch.exp2(e)) & (top > 0)).double()
        unit = torch.exp2(torch.clamp(e - 2, -127, 127))[:, None]
        a = v.abs() / unit
        low, high = torch.bucketize(a, edges), torch.bucketize(a, edges, right=True)
        # on the border of two codes: the even one
        code = torch.where(low % 2 == 0, low, high)
        out[:, b:b + 32] = torch.copysign(grid[code], v) * unit
    return out


def _matmul_exact(s, c):
    q = _nearest_exact(s["x"])
    out = {}
    for i, (w, ws) in enumerate(s["w"]):
        y = torch.matmul(q, _decode_exact(w, ws, c["in"]).t().contiguous())
        out["y%d" % i] = y + s["bias"].double()[None, :] if s["bias"] is not None else y
    return out


def _moe_exact(s, c):
    x = s["x"].double()
    logits = torch.matmul(s["router"].double(), x.t().contiguous()).t().cpu().numpy()
    if c["score"] == "softmax":
        lse = np.log(np.exp(logits - logits.max(1)[:, None]).sum(1)) + logits.max(1)
        score = np.exp(logits - lse[:, None])
    elif c["score"] == "sigmoid":
        score = 0.5 * (1.0 + np.tanh(0.5 * logits))
    else:
        score = np.sqrt(np.logaddexp(0.0, logits))
    key = score.copy()
    if s["bias"] is not None:
        key += s["bias"].cpu().double().numpy()[None, :]
    t, n = key.shape
    rows = np.arange(t)[:, None]
    if c["groups"] > 1:
        per = n // c["groups"]
        best = np.sort(key.reshape(t, c["groups"], per), axis=2)[:, :, per - min(per, c["group_top"]):].sum(2)
        kept = np.argsort(-best, axis=1, kind="stable")[:, :c["top_groups"]]
        allowed = np.zeros((t, c["groups"]), bool)
        allowed[rows, kept] = True
        key[~np.repeat(allowed, per, axis=1)] = -np.inf
    ids = np.argsort(-key, axis=1, kind="stable")[:, :c["top"]]
    w = score[rows, ids]
    if c["renorm"]:
        w = w / w.sum(1)[:, None]
    w = w * c["scale"]
    d, f = c["embd"], c["ff"]
    takes = {}
    for i in range(t):
        for e, v in zip(ids[i].tolist(), w[i].tolist()):
            takes.setdefault(e, []).append((i, v))
    for e in range(c["experts"], c["experts"] + c["shared"]):
        takes[e] = [(i, 1.0) for i in range(t)]
    y = torch.zeros(t, d, dtype=torch.float64, device="cuda")
    for e, pairs in takes.items():
        tok = torch.tensor([i for i, _ in pairs], device="cuda")
        v = torch.tensor([v for _, v in pairs], dtype=torch.float64, device="cuda")
        mine = x[tok].t().contiguous()
        part = {}
        for name, r in (("gate", f), ("up", f), ("down", d)):
            at = slice(e * r, (e + 1) * r)
            part[name] = _decode_exact(s[name][0][at], s[name][1][at], f if name == "down" else d)
        g, u = torch.matmul(part["gate"], mine), torch.matmul(part["up"], mine)
        if c["clamp"] > 1e-6:
            g, u = torch.clamp(g, max=c["clamp"]), torch.clamp(u, min=-c["clamp"], max=c["clamp"])
        h = g * torch.sigmoid(g) * u * v[None, :]
        y.index_add_(0, tok, torch.matmul(part["down"], h).t().contiguous())
    return {"out": y, "ids": ids.astype(np.int32), "weights": w}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "roundtrip":
        return {"values": _nearest_exact(s["x"])}
    return (_moe_exact if case["kind"] == "moe" else _matmul_exact)(s, case)
