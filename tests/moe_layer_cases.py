"""Layers for each kernel of the 4-bit mixture of experts: which kernels take them is
checked in test_moe_layer_launch.py, what comes out in test_gpu_moe_layer_sizes.py."""
#: (pieces of K a wavefront holds the terms of, 0: more than fit; terms of x; terms of h;
#: experts a lane holds the keys of in the choice's own launch, None: the up kernel makes it)
CASES = [
    ((1, 3, 3, None), dict(t=1, embd=513, ff=40)),
    ((1, 3, 2, None), dict(t=8, embd=1537, ff=33, ky="f16", shared=1)),
    ((1, 2, 2, None), dict(t=2, embd=4095, ff=24, kx="f16", ky="bf16", kr="bf16")),
    ((1, 1, 3, 4), dict(t=9, embd=2049, ff=50, kx="bf16", kr="f32", experts=256, k=3, score=1, bias=True)),
    ((1, 1, 2, 0), dict(t=2, embd=260, ff=70, kx="bf16", ky="bf16", experts=257, k=4)),
    ((1, 3, 3, 0), dict(t=11, embd=100, ff=20, experts=600, k=7, groups=6, top_groups=3, group_top=2, score=2,
                        bias=True, scale=1.5)),
    ((2, 3, 3, None), dict(t=3, embd=4097, ff=36, shared=1)),
    ((2, 2, 2, 4), dict(t=19, embd=5000, ff=20, kx="f16", ky="f16", kr="f16", experts=5, k=2, clamp=3.0)),
    ((2, 1, 2, 4), dict(t=32, embd=8192, ff=16, kx="bf16", ky="bf16", kr="bf16", experts=3, k=2)),
    ((0, 3, 3, None), dict(t=2, embd=8193, ff=40)),
    ((0, 2, 3, None), dict(t=6, embd=9999, ff=17, kx="f16", experts=4, k=3)),
    ((0, 1, 2, 4), dict(t=25, embd=12800, ff=16, kx="bf16", ky="bf16", experts=3, k=1, shared=1)),
    # long rows of h, one of which ends inside a step; every token at the same experts
    ((1, 3, 3, None), dict(t=5, embd=40, ff=5000, experts=3, k=1)),
    ((1, 3, 2, 4), dict(t=32, embd=64, ff=2050, experts=2, k=2, ky="bf16")),
    ((1, 3, 3, 4), dict(t=32, embd=164, ff=130, experts=1, k=1, shared=8)),
    # more rows than workgroups take at once
    ((0, 1, 2, None), dict(t=1, embd=8320, ff=16, kx="bf16", ky="bf16", experts=2, k=1)),
]
#: Layers whose down products are summed in parts, up to sixteen: some of them empty, some of
#: one row, tokens that are not finite among them.
PART_CASES = [
    dict(t=32, embd=16, ff=520, experts=8, k=8), dict(t=22, embd=408, ff=1100, experts=8, k=4, kx="bf16", y_gap=3, shared=1),
    dict(t=32, embd=1, ff=600, experts=2, k=2, ky="f16"), dict(t=9, embd=100, ff=2600, experts=5, k=3, kx="f16", ky="bf16"),
    dict(t=32, embd=40, ff=1030, experts=1, k=1, shared=3), dict(t=17, embd=2047, ff=64, experts=16, k=16, ky="bf16", y_gap=1),
]
