"""Where 32-bit keys cannot tell which group stays or which expert is chosen:
biases of both signs that cancel in a group's sum, and equal keys made of other
logits and other biases. The choice is the 64-bit one."""
import numpy as np
import pytest

import serving_ref as R
from test_gpu_route import groups_settled, run

pytestmark = pytest.mark.gpu


def test_two_groups_whose_biases_cancel(hip):
    """The groups count 0.4872955 and 0.4872731; in f32, whose steps at 1000 are
    6e-5, 0.4872437 and 0.4873047."""
    x = np.array([[-1.024, -1.248, -0.99, -1.287]])
    ids, _ = run(hip, x, np.array([1000.0, -1000.0, 1000.0, -1000.0]), 2, 2, 1, 2, score=1)
    assert ids.tolist() == [[0, 1]]


def settled(x, bias, n_group, topk_group, score, size):
    """Rows whose kept groups 64-bit arithmetic settles: a count is of three
    additions of values up to 2 `size`, each off by half of 2^-52 of that, so two
    counts come out up to 6 * 2^-53 * 2 size < 2^-49 size off each other, and the
    scores' last bits less."""
    key = (np.stack([R.scores(l, score) for l in x]) + bias).reshape(len(x), n_group, -1)
    count = np.sort(np.sort(key, axis=2)[:, :, -2:].sum(2), axis=1)
    return count[:, n_group - topk_group] - count[:, n_group - topk_group - 1] > 2.0 ** -48 * size


@pytest.mark.parametrize("score", [0, 1, 2])
@pytest.mark.parametrize("size", [1e2, 1e3, 1e5, 1e6])
@pytest.mark.parametrize("n,groups,topk_group", [(4, 2, 1), (32, 8, 4), (96, 4, 2), (256, 8, 4), (256, 32, 20),
                                                (512, 8, 3), (1024, 16, 5)])
def test_groups_whose_biases_cancel(hip, score, size, n, groups, topk_group):
    """One expert of each group switched on by +size, the others off by -size. The
    logits are a few f32 steps of `size` apart, so that the counts are, too."""
    rng = np.random.default_rng(n + groups + int(size) + score)
    n_tok, per = 150, n // groups
    bias = np.full(n, -size)
    bias[np.arange(groups) * per + rng.integers(0, per, groups)] = size
    x = rng.normal(0, 1, (n_tok, 1)) + rng.normal(0, min(1.0, size * 2.0 ** -21), (n_tok, n))
    x = x.astype(np.float32).astype(np.float64)
    keep = settled(x, bias, groups, topk_group, score, size)
    assert keep.sum() > 0.9 * n_tok
    run(hip, x[keep], bias, min(6, topk_group * per), groups, topk_group, 2, score=score)


@pytest.mark.parametrize("score", [0, 1, 2])
def test_groups_of_biases_of_every_size(hip, score):
    """A group of large biases among groups of small ones: the border lies between
    groups whose own sums are exact to little."""
    rng = np.random.default_rng(40 + score)
    for n, groups, topk_group in ((32, 8, 4), (256, 8, 5), (512, 16, 3)):
        x = rng.normal(0, 1.5, (400, n)).astype(np.float32).astype(np.float64)
        for _ in range(3):
            bias = rng.normal(0, 1, n) * 10.0 ** rng.integers(-3, 7, n)
            bias[rng.random(n) < 0.2] = -1e4
            bias = bias.astype(np.float32).astype(np.float64)
            keep = settled(x, bias, groups, topk_group, score, np.abs(bias).max())
            run(hip, x[keep], bias, 6, groups, topk_group, 2, score=score)
            run(hip, x[keep], bias, 6, groups, topk_group, 1, score=score)


@pytest.mark.parametrize("groups", [(1, 1, 1), (8, 4, 2), (8, 4, 1)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_sums_beyond_f32(hip, groups, sign):
    """Keys near f32's largest: two of them add up to inf in 32 bits."""
    rng = np.random.default_rng(60)
    x = rng.normal(0, 1.5, (50, 64))
    bias = sign * (2e38 + 1e38 * rng.random(64))
    keep = groups_settled(x.astype(np.float32).astype(np.float64), bias.astype(np.float32).astype(np.float64),
                          *groups, 1)
    run(hip, x[keep], bias, 6, *groups, score=1)


@pytest.mark.parametrize("score", [0, 1, 2])
@pytest.mark.parametrize("groups", [(1, 1, 1), (8, 4, 2), (8, 4, 1)])
@pytest.mark.parametrize("n", [64, 128, 256, 1000])
def test_close_keys_of_other_logits_and_biases(hip, score, groups, n):
    """The odd experts' logits lie 1.5 higher, and their biases make up for it to
    within an f32 step of the key: the same key or a neighbour, of another logit
    and another bias."""
    rng = np.random.default_rng(n + score)
    low = np.repeat(rng.normal(0, 0.5, n // 2), 2)  # pairs
    x = np.stack([low + 1.5 * (np.arange(n) % 2)] * 20)
    x[10:] += rng.integers(0, 2, (10, n)) * 2.0 ** -22
    x = x.astype(np.float32).astype(np.float64)
    s = R.scores(x[0], score)
    bias = np.zeros(n)
    bias[1::2] = s[::2] - s[1::2] + rng.integers(-1, 2, n // 2) * 2.0 ** -24
    bias = bias.astype(np.float32).astype(np.float64)
    keep = groups_settled(x, bias, *groups, score)
    assert keep.sum() >= 10
    run(hip, x[keep], bias, 8, *groups, score=score)
