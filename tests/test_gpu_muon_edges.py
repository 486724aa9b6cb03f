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
