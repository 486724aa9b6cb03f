"""The Muon step at its edges: momenta without parameters, updates of few directions, many steps, norms far below eps."""
import math

import pytest
import torch

from test_gpu_muon import allowed, matrix, off, optim, polar  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("where", [0, 1, 2, "all"], ids=str)
@pytest.mark.parametrize("shape", [(40, 90), (130, 200), (200, 130), (2, 300, 1000)], ids=str)
def test_momenta_without_parameters(optim, shape, where):  # noqa: F811
    """They are updated, wherever they stand in the list, and the other entries are what they are without them."""
    alone = [where == "all" or i == where for i in range(3)]
    gs, ms = [matrix(*shape, seed=i) for i in range(3)], [matrix(*shape, seed=10 + i) for i in range(3)]
    ps = [None if a else matrix(*shape, seed=20 + i) for i, a in enumerate(alone)]
    kept = [i for i in range(3) if not alone[i]]
    want_p, want_m = [ps[i].clone() for i in kept], [ms[i].clone() for i in kept]
    if kept:
        optim.muon_step(want_p, [gs[i] for i in kept], want_m, lr=0.1)
    first = [m.clone() for m in ms]
    optim.muon_step(ps, gs, ms, lr=0.1, momentum=0.95)
    for i in range(3):
        # (two roundings, one where they are fused)
        assert off(ms[i], (first[i].double() * 0.95 + gs[i]).cpu()) <= 2.0 ** -23
    for k, i in enumerate(kept):
        assert torch.equal(ms[i], want_m[k])
        # (another split of the depth in a launch of more entries: both are as far off the formula's as they may be)
        rate = 0.1 * math.sqrt(max(1.0, shape[-2] / shape[-1]))
        size = math.sqrt(min(shape[-2:]) * math.prod(shape[:-2]))    # of an orthogonalised stack: singular values of 0.68 to 1.21
        assert float((ps[i] - want_p[k]).norm()) <= 2 * rate * 1.21 * size * allowed(torch.float32) + float(want_p[k].norm()) * 2.0 ** -22


def directions(rows, cols, rank, seed=0):
    """A matrix of exactly ``rank`` directions: products of whole numbers, which fp32 holds; or a few rows over and over."""
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randint(-99, 100, s, generator=g).float()  # noqa: E731
    return (n(rows, rank) @ n(rank, cols)).cuda()


def repeated(rows, cols, rank, seed=0):
    return matrix(rank, cols, seed=seed).repeat(rows // rank, 1)


@pytest.mark.parametrize("steps", [5, 6, 8, 10, 12, 14, 16])
@pytest.mark.parametrize("make", [directions, repeated], ids=lambda f: f.__name__)
@pytest.mark.parametrize("shape", [(16, 1001, 1), (300, 8, 1), (32, 500, 4), (48, 333, 2), (64, 1000, 8), (1500, 64, 1)], ids=str)
def test_few_directions_and_many_steps(optim, shape, make, steps):  # noqa: F811
    """Short sides: what a matrix has no direction for stays nothing, however often that is multiplied by 3.4445."""
    rows, cols, rank = shape
    u = make(rows, cols, rank) if rows < cols else make(cols, rows, rank).t().contiguous()
    # X's own rounding.  Before it all is fp64: Q's roundings, 2^-53 of 3.4445^16 times the length of its sums; and the lift of
    # 2^-48, relative to a small direction's square: the smallest of these is a fifth of the norm or more
    bound = 2.0 ** -24 + 3.4445 ** steps * 2.0 ** -53 * 64 + 2.0 ** -48 * 100
    if steps <= 5:
        # fp32: Q's roundings, each 2^-24 of a row's share of 3.4445^5 at most, over m rows in the norm; and m sums' in each of them,
        # independent and uniform in half a step: 0.58 m; X is 2 / 3 of u in norm or more
        m = min(rows, cols)
        bound += 3.4445 ** steps * 2.0 ** -24 * (math.sqrt(m) + 0.58 * m) * 1.5
    assert off(optim.orthogonalize(u, steps=steps), polar(u, steps)) <= bound


@pytest.mark.parametrize("steps", [5, 8, 12, 16])
@pytest.mark.parametrize("shape", [(16, 1001), (64, 300), (40, 65536), (65536, 3), (50, 64)], ids=str)
def test_singular_values_stay_in_range(optim, shape, steps):  # noqa: F811
    """One direction and its roundings to fp32, which many steps bring up too: the polynomial's largest value is 1.2024 (of singular
    values from 0 to 1, and of its own)."""
    g = torch.Generator().manual_seed(3)
    u = (torch.randn(shape[0], 1, generator=g) @ torch.randn(1, shape[1], generator=g)).cuda()
    x = optim.orthogonalize(u, steps=steps).double()
    assert float(torch.linalg.matrix_norm((x if shape[0] <= shape[1] else x.t()) @ (x.t() if shape[0] <= shape[1] else x), 2)) <= 1.21 ** 2


@pytest.mark.parametrize("steps", [1, 5, 8, 12, 16])
@pytest.mark.parametrize("eps", [1e-30, 1e-7, 1.0])
@pytest.mark.parametrize("shape", [(3, 16), (40, 64), (64, 100), (65, 100), (200, 130)], ids=str)
def test_zeros_stay_zeros(optim, shape, eps, steps):  # noqa: F811
    assert not optim.orthogonalize(torch.zeros(shape, device="cuda"), steps=steps, eps=eps).any()
    p, m = matrix(*shape), torch.zeros(shape, device="cuda")
    want = p.clone()
    optim.muon_step([p], [torch.zeros_like(p)], [m], lr=0.1, steps=steps, eps=eps)
    assert torch.equal(p, want) and not m.any()


@pytest.mark.parametrize("steps", [1, 5, 16])
@pytest.mark.parametrize("norm", [1e-1, 1e-6, 1.001e-7, 1e-7, 1e-9, 1e-12, 1e-16, 1e-25])
@pytest.mark.parametrize("shape", [(20, 50), (65, 100), (300, 130), (512, 768)], ids=str)
def test_norms_below_eps(optim, shape, norm, steps):  # noqa: F811
    """X = u / (|u| + eps) is then small throughout, and as near to 64 bits, relative to itself, as any other."""
    u = matrix(*shape)
    u *= norm / float(u.double().norm())
    # (the bounds of the formula's own tests)
    assert off(optim.orthogonalize(u, steps=steps), polar(u, steps)) <= allowed(u.dtype) * (1 if steps < 16 else 20)


def test_norms_of_a_stack(optim):  # noqa: F811
    """Each matrix has its own, in entries of several matrices and shapes, and beside one that is zero or not finite."""
    us = [matrix(5, 96, 70), matrix(70, 200), matrix(3, 130, 100)]
    scale = [torch.tensor([1.0, 1e-9, 0.0, 1e-14, 1e-5]), torch.tensor(1e-11), torch.tensor([1e-20, math.inf, 3.0])]
    us = [u * s.cuda()[..., None, None] for u, s in zip(us, scale)]
    us[2][1] = math.inf
    for u, x in zip(us, optim.orthogonalize(us)):
        for a, b in zip(u.view(-1, *u.shape[-2:]), x.view(-1, *u.shape[-2:])):
            if not a.isfinite().all():
                assert b.isnan().all()
            elif not a.any():
                assert not b.any()
            else:
                assert off(b, polar(a)) <= allowed(u.dtype)
