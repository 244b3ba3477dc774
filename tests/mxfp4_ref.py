"""Plain 64-bit implementations of the 4-bit floating-point entry points, from their
definitions in include/rsllm_hip.h."""
import numpy as np

import serving_ref as R

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def row_bytes(n):
    return (n + 127) // 128 * 64


def scale_bytes(n):
    return (n + 511) // 512 * 16


def quantize(x):
    """Codes and scales of rows of 64-bit values, as the quantiser lays them out."""
    n, k = x.shape
    codes, scales = np.zeros((n, row_bytes(k)), np.uint8), np.zeros((n, scale_bytes(k)), np.uint8)
    mid = (GRID[1:] + GRID[:-1]) / 2
    for r in range(n):
        for b in range((k + 31) // 32):
            v = x[r, 32 * b:32 * b + 32]
            if not np.isfinite(v).all():
                scales[r, b] = 255
                continue
            top = np.abs(v).max()
            s = 127 + max(-127, int(np.frexp(top)[1]) - 3) if top > 0 else 0
            scales[r, b] = s
            for i, a in enumerate(v):
                m = abs(a) * 2.0 ** (127 - s)
                c = int((m > mid).sum())
                if c < 7 and m == mid[c] and c % 2:  # halfway: the even one of c and c + 1
                    c += 1
                j = 32 * b + i
                codes[r, j // 2] |= (c | (8 if np.signbit(a) else 0)) << (4 * (j % 2))
    return codes, scales


def values(codes, scales, k):
    """Rows of codes as 64-bit values."""
    c = np.stack([codes & 15, codes >> 4], 2).reshape(len(codes), -1)[:, :k]
    v = np.where(c >= 8, -1.0, 1.0) * GRID[c & 7]
    s = scales.astype(np.int64)
    unit = np.where(s == 255, np.nan, 2.0 ** (s - 127.0))
    return v * np.repeat(unit, 32, axis=1)[:, :k]


def random_rows(rng, n, k, low=118, high=124, garbage=True):
    """A matrix of random codes and scales; what stands behind its rows is garbage."""
    codes = rng.integers(0, 256, (n, row_bytes(k))).astype(np.uint8)
    scales = np.full((n, scale_bytes(k)), 255, np.uint8)
    blocks = (k + 31) // 32
    scales[:, :blocks] = rng.integers(low, high + 1, (n, blocks))
    if not garbage:
        clear_tail(codes, k)
    return codes, scales


def clear_tail(codes, k):
    if k % 2:
        codes[:, k // 2] &= 15
    codes[:, (k + 1) // 2:] = 0


def product(x, w, bias):
    """(out, the sum of the terms' magnitudes) of 64-bit matrices."""
    with np.errstate(invalid="ignore"):
        y, size = x @ w.T, np.abs(x) @ np.abs(w).T
    if bias is not None:
        y, size = y + bias, size + np.abs(bias)
    return y, size


def rounding(want, kind):
    """How far one rounding to `kind` is off."""
    return np.abs(want) * R.HALF_STEP[kind] + R.TINY_STEP[kind]


def moe(x, router, bias, gate, up, down, n_expert, n_shared, k, n_group, topk_group, group_top, score, renorm,
        scale, clamp, out_kind):
    """ids, weights, out in 64 bits and how far out may be off. gate, up, down: lists of
    64-bit matrices, the shared experts' behind the others.

    The bound: a product's terms are exact in f32 accumulation (24 bits of x, or of h
    cut to 24 or 16, times two); a sum of n terms takes n / 32 steps of the matrix cores
    and some joins, each off by at most 2^-23 of the terms' magnitudes S: (n / 32 + 40)
    2^-23 S. h = silu(g) u: |silu'| < 1.1, and 2^-20 of itself for the exponential, the
    division and the products; then cut to terms of 8 bits each."""
    with np.errstate(all="ignore"):
        # (a sum in one order for every expert: equal rows are equal)
        logits = np.stack([(row * router).sum(1) for row in x])
    ids, weights = R.route(logits, bias, k, n_group, topk_group, group_top, score, renorm, scale)
    y, err = np.zeros(x.shape), np.zeros(x.shape)
    n_tok, embd = x.shape
    ff = gate[0].shape[0]
    cut = 2.0 ** -24 if out_kind == "f32" else 2.0 ** -16
    for t in range(n_tok):
        slots = [(e, w) for e, w in zip(ids[t], weights[t]) if e >= 0 and np.float32(w) != 0]
        slots += [(n_expert + j, 1.0) for j in range(n_shared)]
        total = np.zeros(embd)
        for e, w in slots:
            with np.errstate(all="ignore"):
                g, u = gate[e] @ x[t], up[e] @ x[t]
                step = (embd / 32 + 40) * 2.0 ** -23
                eg, eu = step * (np.abs(gate[e]) @ np.abs(x[t])), step * (np.abs(up[e]) @ np.abs(x[t]))
                if clamp > 1e-6:
                    g, u = np.minimum(g, clamp), np.clip(u, -clamp, clamp)
                s = g / (1.0 + np.exp(-g))
                h = s * u
                eh = 1.1 * eg * (np.abs(u) + eu) + np.abs(s) * eu + np.abs(h) * (2.0 ** -20 + cut)
                y[t] += w * (down[e] @ h)
                err[t] += w * (np.abs(down[e]) @ eh)
                total += w * (np.abs(down[e]) @ np.abs(h))
        err[t] += (len(slots) * ff / 32 + 40) * 2.0 ** -23 * total
        if not np.isfinite(x[t]).all():
            y[t] = np.nan
    return ids, weights, y, err + rounding(y, out_kind)
