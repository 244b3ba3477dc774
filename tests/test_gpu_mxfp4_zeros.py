"""Decoding 4-bit rows keeps the sign of a zero, in every type and at any alignment."""
import numpy as np
import pytest
import torch

import mxfp4_ref as M
import serving_ref as R
from test_gpu_mxfp4 import run_dequantize

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("k,gap", [(64, 0), (64, 1), (77, 3), (256, 8)])
def test_zeros_keep_their_signs(hip, kind, k, gap):
    rng = np.random.default_rng(k)
    codes, scales = M.random_rows(rng, 5, k, 0, 254)
    codes[:3] &= 0x88
    got = run_dequantize(hip, codes, scales, k, kind, k + gap)[:, :k]
    with np.errstate(over="ignore"):
        want = torch.from_numpy(M.values(codes, scales, k)).float().to(R.TORCH[kind])
    assert (torch.signbit(want) & (want == 0)).any()
    assert torch.equal(torch.signbit(got), torch.signbit(want)) and torch.equal(got, want)
