"""The launches of projections whose weights are held in 4 bits, and the workspace that is reserved for them: what a launch
leaves of a split depth has to fit, whatever the type, the direction, the adapters beside it and the boundaries of the rows."""
import ctypes
import random

import pytest
import torch

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}

# fp32, rows on 16-byte boundaries: whole tiles of a split depth and a few rows behind them, which rows off the boundaries would
# be planned without
SPLIT = [(769, 9216, 4096, 0), (784, 8192, 4096, 0), (769, 8192, 8192, 0), (521, 5120, 4096, 0), (520, 3968, 4096, 23), (773, 7488, 4096, 0),
         (649, 2368, 4096, 0)]


def fits(capi, T, K, N, G, dtype, backward, aligned):
    launches, room = capi.mx4_plan(T, K, N, G, dtype, backward, aligned)
    assert sum(rows for rows, _, _ in launches) == T
    written = max([splits * rows * (K if backward else N) * 4 for rows, _, splits in launches if splits > 1], default=0)
    assert written <= room[0], (T, K, N, G, dtype, backward, aligned, launches, room)
    return launches, room


def workspace(capi, T, K, N, dtype, backward):
    need = ctypes.CDLL(capi.lib()._name)["cp4_mx4_backward_workspace_bytes" if backward else "cp4_mx4_forward_workspace_bytes"]
    need.argtypes, need.restype = [ctypes.c_size_t, ctypes.c_uint, ctypes.c_uint, ctypes.c_int], ctypes.c_size_t
    return need(T, K, N, list(DTYPES.values()).index(dtype))


@pytest.mark.parametrize("T,K,N,G", SPLIT)
def test_partial_sums_of_fp32_prompts_fit(T, K, N, G):
    from paralleltnnlayers_amd import capi
    launches, _ = fits(capi, T, K, N, G, torch.float32, False, True)
    assert len(launches) == 2 and launches[0][2] > 1, "the size stands for a split depth with rows left over"
    assert all(fits(capi, T, K, N, G, torch.float32, back, aligned) for back in (False, True) for aligned in (False, True))


@pytest.mark.parametrize("dtype", list(DTYPES), ids=str)
def test_partial_sums_fit(dtype):
    """Sizes from a token to thousands, many of them a few rows beyond whole tiles."""
    from paralleltnnlayers_amd import capi
    rng = random.Random(dtype)
    size = lambda low, high: int(low * (high / low) ** rng.random())  # noqa: E731
    split = 0
    for i in range(6000):
        T = 128 * rng.randint(2, 16) + rng.randint(0, 33) if i % 2 else size(1, 9000)
        K, N = ((n + 63) // 64 * 64 if rng.random() < 0.6 else n for n in (size(1, 16384), size(1, 16384)))
        G = rng.choice([0, 0, 1, 8, 23, 200])
        for backward in (False, True):
            for aligned in (False, True):
                launches, room = fits(capi, T, K, N, G, DTYPES[dtype], backward, aligned)
                split += any(s > 1 for _, _, s in launches)
            if not G:
                assert sum(room) == workspace(capi, T, K, N, DTYPES[dtype], backward)
    assert split > 3000


def test_plan_query_refuses():
    from paralleltnnlayers_amd import capi
    for bad in (dict(K=0), dict(N=(1 << 22) + 1), dict(T=(1 << 26) + 1), dict(G=65536)):
        with pytest.raises(capi.Cp4Error):
            capi.mx4_plan(**{**dict(T=4, K=8, N=8), **bad})
    L, launches, room = capi.lib(), (capi.AdapterLaunch * 2)(), (ctypes.c_size_t * 2)()
    n = [ctypes.c_size_t(4), ctypes.c_uint(8), ctypes.c_uint(8), ctypes.c_uint(0), 0, 0, 1]
    assert L.cp4_mx4_plan_query(*n, None, room) == L.cp4_mx4_plan_query(*n, launches, None) == capi.ERR_NULL_POINTER
    assert capi.mx4_plan(0, 8, 8) == ([], (0, 0))


@pytest.mark.gpu
@pytest.mark.parametrize("T,K,N,G", SPLIT)
def test_fp32_prompts_against_64_bits(T, K, N, G):
    """Sampled rows, those at the launches' ends among them, y and dx."""
    import paralleltnnlayers_amd as cp4
    from paralleltnnlayers_amd import capi
    from test_gpu_adapter import check, formula, ids_of
    cp4.lib()
    launches, _ = fits(capi, T, K, N, G, torch.float32, False, True)
    gen = torch.Generator(device="cuda").manual_seed(T + K)
    n = lambda *s, std=1.0: torch.randn(*s, device="cuda", generator=gen) * std  # noqa: E731
    q = cp4.mx4_quantize(n(N, K, std=K ** -0.5))
    x, dy, bias, R = n(T, K), n(T, N), n(N), 16
    A, B = n(max(G, 1), R, K, std=K ** -0.5), n(max(G, 1), N, R, std=R ** -0.5)
    ids = ids_of("runs", T, G, torch.Generator().manual_seed(T)).cuda() if G else torch.full((T,), -1, dtype=torch.int32, device="cuda")
    if G:
        y, dx = cp4.adapter_forward(x, q, A, B, ids, bias=bias), cp4.adapter_backward(dy, None, q, A, B, ids, want_factors=False)[0]
    else:
        y, dx = cp4.mx4_linear(x, q, bias), cp4.mx4_linear_backward(dy, q)
    main = launches[0][0]
    rows = {t for t in [*range(0, T, 97), *range(main - 3, main + 3), *range(T - 20, T)] if 0 <= t < T}
    rows = torch.tensor(sorted(rows), device="cuda")
    d = dict(x=x[rows], dy=dy[rows], W=cp4.mx4_dequantize(q), A=A, B=B, ids=ids[rows], bias=bias)
    want = formula(d, "f32", scale=False)
    for name, got in (("y", y), ("dx", dx)):
        value, bound = want[name]
        check(got[rows], (value.cpu(), bound.cpu()), name)
