"""Which kernel the int8 product launches, and what it asks of the runtime first: on
the host, with no kernel run."""
import re

import hip_recorder
from int8_cases import CASES, TILES

CALL = """
def go(t, k, n):
    rb = B.int8_row_bytes(k)
    B.matmul_int8_prequant_dev(4096, t * n, n, 4096, n * rb, 4096, n, 0, 0, 4096, t * rb, 4096, t, 0, 0, t, k, n)
    return rec.rec_take().decode()
"""


def tile(name):
    """Channels x tokens of a kernel, from its (mangled) template arguments."""
    n = [int(v) for v in re.findall(r"Li(\d+)E", name)]
    if "I8Tile" in name:
        wm, wn, _, mf, nf, _ = n
    else:
        wm, wn, mf, nf = n[:4]
    return 16 * mf * wm, 16 * nf * wn


def test_every_kernel_is_reached(tmp_path):
    """The sizes that test_gpu_int8_tiles.py compares go to the kernels they stand
    for, and no kernel is without some."""
    out = hip_recorder.run(tmp_path, CALL + f"""
for i in range(rec.rec_kernels()):
    name = rec.rec_kernel(i).decode()
    if any(k in name for k in ("k_i8_tile", "k_i8_big", "k_i8_wide")):
        print("has", name)
for t, k, n in {[c[1:] for c in CASES]!r}:
    print("ran", go(t, k, n))
""").split("\n")
    has = {tile(line) for line in out if line.startswith("has")}
    ran = [tile(line) for line in out if line.startswith("ran")]
    assert has == set(TILES)
    assert ran == [c[0] for c in CASES]


def test_a_refused_attribute_is_asked_for_again(tmp_path):
    """A runtime that cannot set a kernel's LDS size fails that call alone: the next
    one asks again."""
    sizes = [sizes[0] for sizes in TILES.values()]
    out = hip_recorder.run(tmp_path, CALL + f"""
for t, k, n in {sizes!r}:
    rec.rec_fail(1)
    try:
        go(t, k, n)
        print("launched")
    except B.Error as e:
        print("refused")
    try:
        print(go(t, k, n))
    except B.Error as e:
        print("refused again")
""").split("\n")[:-1]
    assert out[::2] == ["refused"] * len(sizes)
    assert [tile(o) for o in out[1::2] if o != "refused again"] == list(TILES)


def test_each_device_is_asked(tmp_path):
    """The LDS size is a kernel's on one device: after rsllm_hip_init of another it is
    asked for there, too, and once on each."""
    sizes = [sizes[0] for sizes in TILES.values()]
    out = hip_recorder.run(tmp_path, CALL + f"""
for device in (0, 1, 0, 1):
    B.init(device)
    rec.rec_set()
    for t, k, n in {sizes!r}:
        go(t, k, n)
    print(rec.rec_set())
""").split()
    assert out == [str(len(sizes)), str(len(sizes)), "0", "0"]
