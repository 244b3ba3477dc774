"""Plain 64-bit implementations of the routing, int8-product and log-probability
entry points, one row at a time, from their definitions in include/rsllm_hip.h."""
import numpy as np
import torch

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GGML = {"f32": 0, "f16": 1, "bf16": 30}
#: the farthest a rounding is off, relative to the value
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
#: and where the type's numbers get no denser
TINY_STEP = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}


def as_type(a, kind):
    """numpy values rounded to `kind`: (the CPU tensor, its values in 64 bits)."""
    t = torch.from_numpy(np.asarray(a, np.float32)).to(TORCH[kind])
    return t, t.double().numpy()


def strided(t, stride):
    """The rows of t in a buffer where they lie `stride` elements apart; what
    lies between them is NaN. (buffer, elements from the first to the last.)"""
    n, m = t.shape
    buf = torch.full((n, stride), float("nan"), dtype=t.dtype)
    buf[:, :m] = t
    return buf, (n - 1) * stride + m if n else 0


def _exp_diff(l, m):
    with np.errstate(all="ignore"):
        return np.where(l == m, 1.0, np.exp(l - m))


def scores(l, kind):
    """64-bit scores of one row (those of experts never chosen mean nothing)."""
    with np.errstate(all="ignore"):
        if kind == 0:
            live = l[l > -np.inf]
            if not live.size:
                return np.zeros_like(l)
            return _exp_diff(l, live.max()) / _exp_diff(live, live.max()).sum()
        if kind == 1:
            return 1.0 / (1.0 + np.exp(-l))
        return np.sqrt(np.maximum(l, 0.0) + np.log1p(np.exp(-np.abs(l))))


def route(logits, bias, k, n_group, topk_group, group_top, score, renorm, scale):
    """ids [n_tok, k] and weights in 64 bits."""
    n_tok, n = logits.shape
    per = n // n_group
    ids, wts = np.full((n_tok, k), -1, np.int32), np.zeros((n_tok, k))
    for t in range(n_tok):
        l = logits[t]
        s = scores(l, score)
        key = s + bias if bias is not None else s
        place = key if bias is not None else l
        with np.errstate(invalid="ignore"):
            live = (l > -np.inf) & (key > -np.inf)
        groups = []
        for g in range(n_group):
            at = [e for e in range(g * per, (g + 1) * per) if live[e]]
            best = sorted((key[e] for e in at), reverse=True)[:group_top]
            if best:
                groups.append((-sum(best), g))
        kept = {g for _, g in sorted(groups)[:topk_group]} if n_group > 1 else {0}
        order = sorted((-place[e], e) for e in range(n) if live[e] and e // per in kept)[:k]
        chosen = [e for _, e in order]
        ids[t, :len(chosen)] = chosen
        w = s[chosen] * np.float64(np.float32(scale))
        if renorm:
            total = s[chosen].sum()
            w = w / total if total != 0 else np.zeros_like(w)
        wts[t, :len(chosen)] = w
    return ids, wts


def quantize(x):
    """Codes (int8) and f32 scales of rows of 64-bit values."""
    codes, scales = np.zeros(x.shape, np.int8), np.zeros(len(x), np.float32)
    for t, row in enumerate(x):
        if not np.isfinite(row).all():
            scales[t] = np.nan
            continue
        d = np.float32(np.abs(row).max() / 127.0)
        scales[t] = d
        if d > 0:
            codes[t] = np.clip(np.rint(row / np.float64(d)), -127, 127)
    return codes, scales


def int8_product(codes, scales, w, wscale, bias):
    """(out, the product before the bias) in 64 bits."""
    p = (codes.astype(np.float64) @ w.astype(np.float64).T) * scales[:, None].astype(np.float64) \
        * wscale[None, :].astype(np.float64)
    return (p if bias is None else p + bias[None, :].astype(np.float64)), p


def logprobs(logits, tokens, n_top):
    """logprob, rank, entropy, top ids, their log-probabilities; and per row the
    largest |l - m| that carries weight (for error bounds)."""
    n_tok, v = logits.shape
    lp, rank, ent = np.full(n_tok, np.nan), np.zeros(n_tok, np.int32), np.zeros(n_tok)
    ids, top = np.full((n_tok, n_top), -1, np.int32), np.full((n_tok, n_top), -np.inf)
    with np.errstate(all="ignore"):
        for t in range(n_tok):
            l = logits[t]
            bad, live = np.isnan(l).any(), l > -np.inf
            m = l[live].max() if live.any() else -np.inf
            e = np.where(live, _exp_diff(l, m), 0.0) if live.any() else np.zeros(v)
            total = e.sum()

            def one(x):
                if bad:
                    return np.nan
                if not live.any():
                    return -np.inf
                return (0.0 if x == m else x - m) - np.log(total)
            if live.any():
                p = e / total
                ent[t] = -(p[p > 0] * np.log(p[p > 0])).sum()
            if bad:
                ent[t] = np.nan
            if tokens is not None and 0 <= tokens[t] < v:
                x = l[tokens[t]]
                lp[t] = one(x)
                rank[t] = 0 if np.isnan(x) else 1 + (l > x).sum()
            order = sorted((-l[i] + 0.0, i) for i in np.flatnonzero(live))[:n_top] if v <= 4096 else \
                [(-l[i], i) for i in _largest(l, n_top)]
            for r, (_, i) in enumerate(order):
                ids[t, r], top[t, r] = i, one(l[i])
            if bad:
                top[t] = np.nan
    return lp, rank, ent, ids, top


def _largest(l, n):
    at = np.flatnonzero(l > -np.inf)
    return at[np.argsort(-l[at], kind="stable")][:n]
