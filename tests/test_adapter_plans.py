"""Every kernel that the adapters' shared projection chooses from, at sizes that it takes them for: each shape of tile in
both directions, with the depth whole and split, fed directly and through registers, the kernel of few rows, and what
whole tiles leave over.  The plans stand beside the sizes, so that a change of the choice cannot leave a kernel without a test."""
import pytest
import torch

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ROWS = None                # the kernel of few rows
R, G = 20, 4

PLANS = [  # 16-bit or fp32, dx or y, T, K, N, launches
    ("16", "y", 65, 65, 72, [(65, (128, 128), 1)]),
    ("16", "y", 513, 4097, 8192, [(512, (128, 128), 1), (1, ROWS, 1)]),
    ("16", "y", 65, 1001, 200, [(65, (128, 128), 4)]),
    ("16", "y", 257, 65, 14336, [(257, (64, 256), 1)]),
    ("16", "y", 2077, 4097, 8192, [(2048, (64, 256), 1), (29, (64, 256), 8)]),
    ("16", "y", 2049, 1001, 4096, [(2048, (64, 256), 1), (1, ROWS, 1)]),
    ("16", "y", 17, 4097, 4097, [(17, (64, 256), 13)]),
    ("16", "y", 3, 1001, 200, [(3, ROWS, 1)]),
    ("16", "y", 3, 4097, 200, [(3, ROWS, 4)]),
    ("16", "y", 65, 512, 200, [(65, (128, 128), 1)]),
    ("16", "y", 513, 2048, 8192, [(512, (128, 128), 1), (1, ROWS, 1)]),
    ("16", "y", 65, 1016, 200, [(65, (128, 128), 4)]),
    ("16", "y", 257, 72, 14336, [(257, (128, 256), 1)]),
    ("16", "y", 257, 8192, 14336, [(257, (128, 256), 3)]),
    ("16", "y", 513, 72, 14337, [(513, (256, 256), 1)]),
    ("16", "y", 2077, 2048, 14337, [(2048, (256, 256), 1), (29, (64, 256), 4)]),
    ("16", "y", 2049, 512, 8192, [(2048, (256, 256), 1), (1, ROWS, 1)]),
    ("16", "y", 257, 4096, 14336, [(257, (256, 256), 2)]),
    ("16", "y", 2077, 8192, 4096, [(2048, (256, 256), 2), (29, (64, 256), 16)]),
    ("16", "y", 513, 8192, 14337, [(512, (256, 256), 2), (1, ROWS, 1)]),
    ("16", "y", 513, 72, 14336, [(513, (64, 256), 1)]),
    ("16", "y", 17, 4096, 4097, [(17, (64, 256), 13)]),
    ("16", "y", 3, 512, 200, [(3, ROWS, 1)]),
    ("16", "y", 3, 4096, 200, [(3, ROWS, 4)]),
    ("16", "dx", 3, 512, 257, [(3, (128, 128), 1)]),
    ("16", "dx", 2049, 2048, 4097, [(2048, (128, 128), 1), (1, (128, 128), 13)]),
    ("16", "dx", 513, 8192, 4097, [(512, (128, 128), 1), (1, (64, 256), 13)]),
    ("16", "dx", 3, 512, 1001, [(3, (128, 128), 4)]),
    ("16", "dx", 1026, 4097, 72, [(1026, (64, 256), 1)]),
    ("16", "dx", 2049, 4096, 4097, [(2048, (64, 256), 1), (1, (64, 256), 13)]),
    ("16", "dx", 3, 1001, 14336, [(3, (64, 256), 56)]),
    ("16", "dx", 2049, 1001, 14336, [(2048, (64, 256), 4), (1, (64, 256), 56)]),
    ("16", "dx", 3, 512, 200, [(3, (128, 128), 1)]),
    ("16", "dx", 2077, 2048, 4096, [(2048, (128, 128), 1), (29, (128, 128), 16)]),
    ("16", "dx", 2049, 2048, 4096, [(2048, (128, 128), 1), (1, (128, 256), 32)]),
    ("16", "dx", 513, 8192, 4096, [(512, (128, 128), 1), (1, (64, 256), 16)]),
    ("16", "dx", 3, 512, 14336, [(3, (128, 128), 56)]),
    ("16", "dx", 2049, 2048, 72, [(2049, (128, 256), 1)]),
    ("16", "dx", 2049, 4096, 4096, [(2048, (128, 256), 1), (1, (64, 256), 16)]),
    ("16", "dx", 3, 512, 1016, [(3, (128, 256), 8)]),
    ("16", "dx", 2049, 4096, 512, [(2049, (256, 256), 1)]),
    ("16", "dx", 2077, 8192, 1016, [(2048, (256, 256), 1), (29, (128, 128), 4)]),
    ("16", "dx", 2049, 8192, 1016, [(2048, (256, 256), 1), (1, (128, 256), 8)]),
    ("16", "dx", 2049, 8192, 4096, [(2048, (256, 256), 1), (1, (64, 256), 16)]),
    ("16", "dx", 130, 8192, 8192, [(130, (256, 256), 8)]),
    ("16", "dx", 2049, 2048, 14336, [(2048, (256, 256), 4), (1, (64, 256), 56)]),
    ("16", "dx", 3, 1016, 14336, [(3, (64, 256), 56)]),
    ("f32", "y", 33, 65, 72, [(33, (128, 128), 1)]),
    ("f32", "y", 700, 4097, 8192, [(512, (128, 128), 1), (188, (64, 256), 5)]),
    ("f32", "y", 257, 1001, 14336, [(256, (128, 128), 1), (1, ROWS, 1)]),
    ("f32", "y", 33, 1001, 200, [(33, (128, 128), 8)]),
    ("f32", "y", 257, 65, 14336, [(257, (64, 256), 1)]),
    ("f32", "y", 700, 4097, 14336, [(512, (64, 256), 1), (188, (64, 256), 3)]),
    ("f32", "y", 513, 1001, 14337, [(512, (64, 256), 1), (1, ROWS, 1)]),
    ("f32", "y", 33, 1001, 4097, [(33, (64, 256), 8)]),
    ("f32", "y", 2049, 4097, 1001, [(2048, (64, 256), 4), (1, ROWS, 4)]),
    ("f32", "y", 3, 1001, 200, [(3, ROWS, 1)]),
    ("f32", "y", 3, 4097, 200, [(3, ROWS, 8)]),
    ("f32", "y", 33, 72, 72, [(33, (128, 128), 1)]),
    ("f32", "y", 700, 2048, 8192, [(512, (128, 128), 1), (188, (64, 256), 5)]),
    ("f32", "y", 257, 512, 14336, [(256, (128, 128), 1), (1, ROWS, 1)]),
    ("f32", "y", 33, 512, 200, [(33, (128, 128), 4)]),
    ("f32", "y", 257, 72, 14336, [(257, (64, 256), 1)]),
    ("f32", "y", 700, 2048, 14336, [(512, (64, 256), 1), (188, (64, 256), 3)]),
    ("f32", "y", 513, 512, 14337, [(512, (64, 256), 1), (1, ROWS, 1)]),
    ("f32", "y", 33, 1016, 4097, [(33, (64, 256), 8)]),
    ("f32", "y", 700, 4096, 8192, [(512, (64, 256), 2), (188, (64, 256), 5)]),
    ("f32", "y", 2049, 4096, 1001, [(2048, (64, 256), 4), (1, ROWS, 4)]),
    ("f32", "y", 3, 512, 200, [(3, ROWS, 1)]),
    ("f32", "y", 3, 2048, 200, [(3, ROWS, 4)]),
    ("f32", "dx", 3, 1001, 200, [(3, (128, 128), 1)]),
    ("f32", "dx", 2049, 2048, 1001, [(2048, (128, 128), 1), (1, (128, 128), 8)]),
    ("f32", "dx", 513, 8192, 1001, [(512, (128, 128), 1), (1, (64, 256), 8)]),
    ("f32", "dx", 3, 512, 257, [(3, (128, 128), 2)]),
    ("f32", "dx", 1026, 4097, 72, [(1026, (64, 256), 1)]),
    ("f32", "dx", 2049, 4096, 1001, [(2048, (64, 256), 1), (1, (128, 128), 8)]),
    ("f32", "dx", 1026, 8192, 1001, [(1024, (64, 256), 1), (2, (64, 256), 8)]),
    ("f32", "dx", 3, 4097, 1001, [(3, (64, 256), 8)]),
    ("f32", "dx", 2049, 1001, 4096, [(2048, (64, 256), 4), (1, (128, 128), 32)]),
    ("f32", "dx", 2049, 1001, 8192, [(2048, (64, 256), 4), (1, (64, 256), 64)]),
    ("f32", "dx", 3, 512, 200, [(3, (128, 128), 1)]),
    ("f32", "dx", 2049, 2048, 1016, [(2048, (128, 128), 1), (1, (128, 128), 8)]),
    ("f32", "dx", 513, 8192, 1016, [(512, (128, 128), 1), (1, (64, 256), 8)]),
    ("f32", "dx", 3, 512, 512, [(3, (128, 128), 4)]),
    ("f32", "dx", 2049, 2048, 72, [(2049, (64, 256), 1)]),
    ("f32", "dx", 2049, 4096, 512, [(2048, (64, 256), 1), (1, (128, 128), 4)]),
    ("f32", "dx", 1026, 8192, 1016, [(1024, (64, 256), 1), (2, (64, 256), 8)]),
    ("f32", "dx", 3, 1016, 8192, [(3, (64, 256), 64)]),
    ("f32", "dx", 2049, 1016, 4096, [(2048, (64, 256), 4), (1, (128, 128), 32)]),
    ("f32", "dx", 1026, 2048, 4096, [(1024, (64, 256), 4), (2, (64, 256), 32)]),
]


def aligned(kind, which, K, N):
    """Whether rows start on 16-byte boundaries: those of x and W, or of dy and W."""
    vec = 4 if kind == "f32" else 8
    return K % vec == 0 and (which == "y" or N % vec == 0)


def plan(kind, which, T, K, N):
    from paralleltnnlayers_amd import capi
    dtype = DTYPES["f32" if kind == "f32" else "bf16"]
    return capi.adapter_plan(T, K, N, R, G, dtype, backward=which == "dx", aligned=aligned(kind, which, K, N))


def test_plans():
    """(on 256 compute units, which is also what is planned for without a device)"""
    for kind, which, T, K, N, want in PLANS:
        assert plan(kind, which, T, K, N) == want, (kind, which, T, K, N)


def test_every_kernel_is_in_the_list():
    have = set()
    for kind, which, T, K, N, launches in PLANS:
        for _, tile, splits in launches:
            have.add((kind, which, aligned(kind, which, K, N), tile, splits > 1))
    tiles = {("16", True): [(128, 128), (128, 256), (64, 256), (256, 256)], ("16", False): [(128, 128), (64, 256)],
             ("f32", True): [(128, 128), (64, 256)], ("f32", False): [(128, 128), (64, 256)]}
    want = {(kind, which, direct, tile, split) for (kind, direct), shapes in tiles.items() for which in ("y", "dx")
            for tile in shapes for split in (False, True)}
    want |= {(kind, "y", direct, ROWS, split) for kind in ("16", "f32") for direct in (False, True) for split in (False, True)}
    want.remove(("16", "dx", True, (64, 256), False))                # (128 x 256 takes its sizes)
    assert have == want
    alone = {(kind, which, launches[1][1]) for kind, which, _, _, _, launches in PLANS if len(launches) == 2}
    assert {("16", "y", ROWS), ("16", "y", (64, 256)), ("16", "dx", (128, 128)), ("16", "dx", (128, 256)), ("16", "dx", (64, 256)),
            ("f32", "y", ROWS), ("f32", "y", (64, 256)), ("f32", "dx", (128, 128)), ("f32", "dx", (64, 256))} <= alone


def test_plan_query_refuses():
    import ctypes
    from paralleltnnlayers_amd import capi
    with pytest.raises(capi.Cp4Error):
        capi.adapter_plan(4, 8, 8, 257, 1)
    L, s = capi.lib(), capi.AdapterShape(T=4, K=8, N=8, R=4, G=1)
    assert L.cp4_adapter_plan_query(ctypes.byref(s), 0, 0, 1, None) == capi.ERR_NULL_POINTER
    assert L.cp4_adapter_plan_query(None, 0, 0, 1, (capi.AdapterLaunch * 2)()) == capi.ERR_NULL_POINTER
    assert capi.adapter_plan(0, 8, 8, 4, 1) == []


CASES = [(dtype, *p) for p in PLANS for dtype in (["f32"] if p[0] == "f32" else ["bf16", "f16"])]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kind,which,T,K,N,launches", CASES, ids=lambda v: None if isinstance(v, list) else str(v))
def test_against_64_bits(dtype, kind, which, T, K, N, launches):
    """Sampled rows, those at the launches' ends among them, within the bounds of the layer's own tests."""
    import paralleltnnlayers_amd as cp4
    from test_gpu_adapter import check, formula, ids_of
    assert plan(kind, which, T, K, N) == launches
    gen = torch.Generator(device="cuda").manual_seed(T + K + N)
    n = lambda *s, std=1.0: (torch.randn(*s, device="cuda", generator=gen) * std).to(DTYPES[dtype])  # noqa: E731
    x, dy, W = n(T, K), n(T, N), n(N, K, std=K ** -0.5)
    A, B = n(G, R, K, std=K ** -0.5), n(G, N, R, std=R ** -0.5)
    ids = ids_of("runs" if T > 64 else "mixed", T, G, torch.Generator().manual_seed(T)).cuda()
    scale, bias = 0.25 + torch.rand(G, device="cuda", generator=gen), torch.randn(N, device="cuda", generator=gen)
    if which == "y":
        got = cp4.adapter_forward(x, W, A, B, ids, scale, bias)
    else:
        got = cp4.adapter_backward(dy, None, W, A, B, ids, scale, want_factors=False)[0]
    main = launches[0][0]
    rows = {t for t in [*range(0, T, 97), *range(main - 3, main + 3), *range(T - 20, T)] if 0 <= t < T}
    rows = torch.tensor(sorted(rows), device="cuda")
    d = dict(x=x[rows], dy=dy[rows], W=W, A=A, B=B, ids=ids[rows], scale=scale, bias=bias)
    value, bound = formula(d, dtype)[which]
    check(got[rows], (value.cpu(), bound.cpu()), which)
