"""Every kernel of the 4-bit product, at sizes that its tile does not divide, against
64-bit sums."""
import pytest

import mxfp4_ref as M
from mxfp4_cases import CASES
from test_gpu_mxfp4 import Product, dev

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("i", range(len(CASES)), ids=["%dx%dx%d-%d-%d-%d" % (*c[0], *c[1:]) for c in CASES])
def test_tile(hip, i):
    _, t, k, n = CASES[i]
    # rows that can be stored four channels at a time, and rows that cannot
    for kind, gap in (("f32", 0), ("bf16", (-n) % 4), ("f16", 1)):
        p = Product(hip, t, k, n, ky=kind, bias=i % 2 == 0, y_gap=gap)
        codes, scales = M.random_rows(p.rng, t, k)
        M.clear_tail(codes, k)
        p.check(p.prequant(dev(codes), dev(scales)), codes, scales)
