"""Which kernels the 4-bit product of float tokens launches: on the host, with no kernel run."""
import re

import hip_recorder
from mxfp4_cases import CASES

FEW = sorted({c[0] for c in CASES if c[0][1] == 16})


def test_one_and_two_tokens_take_one_launch(tmp_path):
    """Of the tiles for few tokens, each with each type; more tokens are quantised first."""
    sizes = [next((t, k, n) for tile, t, k, n in CASES if tile == few and t <= 2) if few != (16, 16, 8) else (1, 2054, 1)
             for few in FEW]
    out = hip_recorder.run(tmp_path, f"""
for i in range(rec.rec_kernels()):
    print("has", rec.rec_kernel(i).decode())
for t, k, n in {sizes + [(3, 4096, 200), (300, 4096, 2048)]!r}:
    for kind in (0, 1, 30):
        B.matmul_mxfp4_dev(4096, t * n, n, 4096, n * B.mxfp4_row_bytes(k), 4096, n * B.mxfp4_scale_bytes(k), 0, 0,
                           4096, t * k, k, 4096, 1 << 40, t, k, n, kind, kind)
        print("ran", *reversed(list(iter(lambda: rec.rec_take().decode(), ""))))
""").split("\n")
    # the kernels whose last template argument is a type of tokens
    has = {line.split()[1] for line in out if re.match(r"has .*k_mx_few.*Lj(0|1|30)E", line)}
    ran = [line.split()[1:] for line in out if line.startswith("ran")]
    assert len(has) == 3 * len(FEW)
    assert {k for names in ran for k in names if k in has} == has
    assert [len(names) for names in ran] == [1] * len(has) + [2] * 6
    assert all("k_mx_quantize" in names[0] for names in ran[len(has):])
