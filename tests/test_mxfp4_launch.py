"""Which kernel the 4-bit product launches, and what it asks of the runtime first: on the
host, with no kernel run."""
import re

import hip_recorder
from mxfp4_cases import CASES, TILES

CALL = """
def go(t, k, n):
    rb, sb = B.mxfp4_row_bytes(k), B.mxfp4_scale_bytes(k)
    B.matmul_mxfp4_prequant_dev(4096, t * n, n, 4096, n * rb, 4096, n * sb, 0, 0, 4096, t * rb, 4096, t * sb,
                                4096, 1 << 40, t, k, n)
    return rec.rec_take().decode()
"""


def tile(name):
    """Channels, tokens and wavefronts along K of a kernel, from its (mangled) template
    arguments."""
    n = [int(v) for v in re.findall(r"Li(\d+)E", name)]
    if "MxFew" in name:
        return 16 * n[0], 16 * n[1], n[2]
    if "MxWide" in name:
        return 32 * n[0], 32 * n[1], 1
    return 16 * n[2] * n[0], 16 * n[3] * n[1], 1


def test_every_kernel_is_reached(tmp_path):
    """The sizes that test_gpu_mxfp4_tiles.py compares go to the kernels they stand for,
    and no kernel is without some."""
    out = hip_recorder.run(tmp_path, CALL + f"""
for i in range(rec.rec_kernels()):
    name = rec.rec_kernel(i).decode()
    if any(k in name for k in ("k_mx_few", "k_mx_big", "k_mx_wide")):
        print("has", name)
for t, k, n in {[c[1:] for c in CASES]!r}:
    print("ran", go(t, k, n))
""").split("\n")
    has = {tile(line) for line in out if line.startswith("has")}
    ran = [tile(line) for line in out if line.startswith("ran")]
    assert has == set(TILES)
    assert ran == [c[0] for c in CASES]


def lds_cases():
    """A size of each kernel that needs more LDS than it gets unasked."""
    return [next(c[1:] for c in CASES if c[0] == t) for t in TILES if t[1] >= 64 and t[2] == 1]


def test_a_refused_attribute_is_asked_for_again(tmp_path):
    """A runtime that cannot set a kernel's LDS size fails that call alone: the next one
    asks again."""
    sizes = lds_cases()
    out = hip_recorder.run(tmp_path, CALL + f"""
for t, k, n in {sizes!r}:
    rec.rec_fail(1)
    for _ in range(2):
        try:
            go(t, k, n)
            print("launched")
        except B.Error as e:
            print("refused")
""").split()
    assert out == ["refused", "launched"] * len(sizes)


def test_each_device_is_asked(tmp_path):
    """The LDS size is a kernel's on one device: after rsllm_hip_init of another it is
    asked for there, too, and once on each."""
    sizes = lds_cases()
    out = hip_recorder.run(tmp_path, CALL + f"""
for device in (0, 1, 0, 1):
    B.init(device)
    rec.rec_set()
    for t, k, n in {sizes!r}:
        go(t, k, n)
    print(rec.rec_set())
""").split()
    assert out == [str(len(sizes)), str(len(sizes)), "0", "0"]
