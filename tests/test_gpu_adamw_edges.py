"""The AdamW step where its arguments are unusual: signs, tiny values, gradients that are not there."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F = np.float32
HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.0)


@pytest.fixture(scope="module")
def optim():
    from paralleltnnlayers_amd import capi, optim
    capi.lib()
    return optim


@pytest.mark.parametrize("most", [0.25, 1.0, 100.0])
@pytest.mark.parametrize("scale", [-1.0, -0.125])
def test_clipping_with_a_negative_grad_scale(optim, scale, most):
    """The norm is a 2-norm whatever the scale's sign, and the step is that of the gradients with their signs turned."""
    gen = torch.Generator().manual_seed(1)
    G = [torch.randn(n, generator=gen).cuda() for n in (5, 300, 5000)]

    def step(grads, scale):
        P = [torch.ones_like(g) for g in grads]
        M = [optim.empty_moments(p) for p in P]
        norm = optim.adamw_step(P, grads, [m for m, _, _ in M], [v for _, v, _ in M], optim.counter(),
                                max_norm=most, grad_scale=scale, **HYPER)
        return [norm, *P, *(m for m, _, _ in M), *(v for _, v, _ in M)]

    got, want = step(G, scale), step([-g for g in G], -scale)        # (a sign is exact)
    assert float(got[0]) > 0
    assert all(torch.equal(a, b) for a, b in zip(got, want))
