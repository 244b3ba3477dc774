"""Which kernels the 4-bit mixture of experts launches, and what it asks of the runtime first:
on the host, with no kernel run."""
import re

import hip_recorder
from moe_layer_cases import CASES

CALL = """
KIND = {"f32": 0, "f16": 1, "bf16": 30}
def go(t, embd, ff, experts=8, k=2, shared=0, groups=1, top_groups=1, group_top=1, score=0, bias=False,
       scale=1.0, clamp=0.0, kx="f32", ky="f32", kr="f32", **_):
    n = experts + shared
    rows, scales = B.mxfp4_row_bytes, B.mxfp4_scale_bytes
    lay = B.MoeMxfp4(router=4096, router_len=experts * embd, dtype_router=KIND[kr], bias=4096 if bias else 0,
                     bias_len=experts if bias else 0, gate=4096, up=4096, gate_up_len=n * ff * rows(embd),
                     gate_scales=4096, up_scales=4096, gate_up_scales_len=n * ff * scales(embd), down=4096,
                     down_len=n * embd * rows(ff), down_scales=4096, down_scales_len=n * embd * scales(ff),
                     n_embd=embd, n_ff=ff, n_expert=experts, n_shared=shared, k=k, n_group=groups,
                     topk_group=top_groups, group_top=group_top, score=score, renormalise=1, scale=scale, clamp=clamp)
    B.moe_mxfp4_dev(lay, 4096, t * embd, embd, 4096, 4096, t * k, 4096, t * embd, embd, 4096, 1 << 40, t,
                    KIND[kx], KIND[ky])
    ran = list(iter(lambda: rec.rec_take().decode(), ""))
    return " ".join(reversed(ran))
"""
NAMES = ("k_moe_in", "k_moe_choose", "k_moe_up", "k_moe_down")


def kernels(line):
    """Names and integer template arguments of the layer's kernels in a line."""
    found = re.findall("(%s)I((?:L[ij]\\d+E)+)E" % "|".join(NAMES), line)
    return [(name, *(int(v) for v in re.findall(r"L[ij](\d+)E", args))) for name, args in found]


def variant(line):
    """The case's variant, from its launches."""
    ran = kernels(line)
    args = {k[0]: k[1:] for k in ran}
    assert [k[0] for k in ran] == [n for n in NAMES if n in args]
    return (*args["k_moe_up"], *args["k_moe_down"], *args.get("k_moe_choose", (None,)))


def test_every_kernel_is_reached(tmp_path):
    out = hip_recorder.run(tmp_path, CALL + f"""
for i in range(rec.rec_kernels()):
    name = rec.rec_kernel(i).decode()
    if any(k in name for k in {NAMES!r}):
        print("has", name)
for c in {[c[1] for c in CASES]!r}:
    print("ran", go(**c))
for kx in KIND:
    for kr in KIND:
        print("types", go(1, 32, 32, kx=kx, kr=kr))
""").split("\n")
    has = {k for line in out if line.startswith("has") for k in kernels(line)}
    ran = {k for line in out if line.startswith(("ran", "types")) for k in kernels(line)}
    # (the routed experts' own kernels have none of these names with these arguments)
    assert ran == has
    assert [variant(line) for line in out if line.startswith("ran")] == [c[0] for c in CASES]


def lds_cases():
    """A layer for each kernel that asks for more LDS than it gets unasked, each after those of
    the layers before it have been granted."""
    seen, cases = set(), []
    for v, c in CASES:
        new = {("up", v[0], v[1]), ("down", v[2])} - seen
        seen |= new
        if new:
            cases.append((len(new), c))
    return cases


def test_a_refused_attribute_is_asked_for_again(tmp_path):
    """A runtime that cannot set a kernel's LDS size fails that call alone: the next one
    asks again."""
    out = hip_recorder.run(tmp_path, CALL + f"""
for new, c in {lds_cases()!r}:
    rec.rec_fail(1)
    for _ in range(2):
        try:
            go(**c)
            print("launched")
        except B.Error as e:
            print("refused")
""").split()
    assert out == ["refused", "launched"] * len(lds_cases())


def test_each_device_is_asked(tmp_path):
    """The LDS size is a kernel's on one device: after rsllm_hip_init of another it is asked
    for there, too, and once on each."""
    cases = lds_cases()
    out = hip_recorder.run(tmp_path, CALL + f"""
for device in (0, 1, 0, 1):
    B.init(device)
    rec.rec_set()
    for new, c in {cases!r}:
        go(**c)
    print(rec.rec_set())
""").split()
    n = str(sum(new for new, _ in cases))
    assert out == [n, n, "0", "0"]


def test_few_rows_and_many_jobs_are_summed_in_parts(tmp_path):
    """Fewer rows than half of the chip takes, with enough for a wavefront to do: parts of the
    down products and a launch that adds them; their workspace counts."""
    sizes = [(32, 64, 2050, True), (22, 408, 2687, True), (32, 2048, 1024, True), (1, 64, 2050, False),
             (3, 408, 128, False), (32, 2064, 1024, False), (32, 4096, 2048, False)]
    out = hip_recorder.run(tmp_path, CALL + f"""
for t, embd, ff, _ in {sizes!r}:
    print(go(t, embd, ff, experts=32, k=8).count("k_moe_sum"))
""").split()
    assert out == [str(int(parts)) for *_, parts in sizes]
