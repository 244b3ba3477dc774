"""The workspace size of the 4-bit expert layer is 0 for a layer whose numbers the call
refuses."""
import pytest

from test_abi_validation_mxfp4 import layer


@pytest.mark.parametrize("kw", [
    dict(n_embd=0), dict(n_embd=65537), dict(n_ff=0), dict(n_ff=65537), dict(n_expert=0), dict(n_shared=9), dict(k=0),
    dict(k=33), dict(k=9), dict(n_group=4, topk_group=1, k=3), dict(n_group=0), dict(n_group=3),
    dict(n_group=4, topk_group=0), dict(n_group=4, topk_group=5), dict(group_top=3)])
def test_no_workspace_for_a_refused_layer(hip, kw):
    assert hip.moe_mxfp4_work_bytes(layer(hip), 3) > 0
    assert hip.moe_mxfp4_work_bytes(layer(hip, **kw), 3) == 0
