"""The 4-bit product of one and two float tokens, which its kernels quantise for themselves,
with each tile and type: the bits of quantising first, and what the definition gives."""
import pytest
import torch

import mxfp4_ref as M
from test_gpu_mxfp4 import Product, dev, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("t,k,n", [(1, 2054, 1), (2, 4096, 200), (1, 9000, 33), (1, 2100, 4282), (2, 4001, 4300),
                                   (1, 258, 1), (2, 1030, 300), (2, 511, 40), (1, 513, 40), (2, 14336, 64)])
def test_tiles_and_types(hip, kind, t, k, n):
    for gap in (0, 1, 8):
        Product(hip, t, k, n, kind, kind, bias=n % 2 == 0, x_gap=gap, y_gap=gap).both()


@pytest.mark.parametrize("t", [1, 2])
@pytest.mark.parametrize("k", [40, 2100])
def test_not_finite_blocks(hip, t, k):
    """A token with an infinity is NaN throughout, the one beside it is itself."""
    p = Product(hip, t, k, 50)
    p.x[t - 1, k - 1] = float("inf")
    p.xt = torch.from_numpy(p.x).float()
    p.d["x"], p.span = rows(p.xt, k)
    p.both()
    assert torch.isnan(p.out[t - 1]).all() and (t == 1 or not torch.isnan(p.out[0]).any())


def test_the_workspace_holds_anything(hip):
    """What stands in the workspace does not matter, whether the call uses it or not."""
    p = Product(hip, 2, 2100, 96, bias=True)
    codes, scales = M.quantize(p.x)
    want = p.prequant(dev(codes), dev(scales))
    for fill in (0, 255):
        p.work.fill_(fill)
        assert torch.equal(p.oneshot(), want)
