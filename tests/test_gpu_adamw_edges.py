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


def in_64_bits(qm, qv, scales):
    """What codes and scales stand for, by the definition."""
    at = torch.arange(qm.numel()) // 256
    m, v, s = qm.cpu().double(), qv.cpu().double(), scales.cpu().double()
    return m * m.abs() / 127.0 ** 2 * s[0][at], (v / 255.0) ** 4 * s[1][at]


# A moment is read with four roundings or fewer (its units' constant, the scale times that, the code's fourth power, their
# product), and is a denormal number below 2^-126, 2^-149 apart.
UNITS, STEP = 4 * 2.0 ** -24, 2.0 ** -149


@pytest.mark.parametrize("top", [3e38, 1e10, 1.5, 0.75, 1e-28, 1e-30, 1e-35, 1e-36, 2e-38])
def test_moments_of_any_scale(optim, top):
    """Blocks of every level, from the largest scales to the smallest: read as in 64 bits, and a second moment above zero
    never as zero."""
    q = torch.arange(256)
    m, v = ((q - 127).clamp(max=127).double() / 127), (q.double() / 255)
    m, v = (m * m.abs() * top).float(), (v ** 4 * top).float()
    v[1:3] = 2.0 ** -149                                             # far below the least level of most of these blocks
    qm, qv, s = optim.empty_moments(torch.empty(256, device="cuda"), 8)
    optim.set_moments([qm], [qv], [s], ([m.cuda()], [v.cuda()]))
    above = v > 0                                                    # (the least levels of the smallest blocks are no numbers)
    assert torch.equal(qv.cpu() > 0, above)
    (a,), (b,) = optim.moment_values([qm], [qv], [s])
    for got, want in zip((a, b), in_64_bits(qm, qv, s)):
        assert ((got.cpu().double() - want).abs() <= UNITS * want.abs() + STEP).all()
    assert torch.equal(b.cpu() > 0, above)
    normal = v >= 2.0 ** -126
    assert torch.equal(qv.cpu()[normal].long(), q[normal])           # (a level comes back as itself)


def test_a_step_without_eps_on_tiny_moments(optim):
    """eps = 0 and gradients that have become zero: the step divides by what the codes still hold."""
    gen = torch.Generator().manual_seed(2)
    n = 512
    v = (0.1 + 0.9 * torch.rand(n, generator=gen)) * 1e-36
    m = v.double().sqrt().float() * (0.5 + torch.rand(n, generator=gen)) * (1 - 2 * torch.randint(0, 2, (n,), generator=gen))
    p = torch.randn(n, generator=gen)
    qm, qv, s = optim.empty_moments(torch.empty(n, device="cuda"), 8)
    optim.set_moments([qm], [qv], [s], ([m.cuda()], [v.cuda()]))
    M, V = in_64_bits(qm, qv, s)
    lr, (b1, b2), t = 1e-3, (0.9, 0.99), 10
    count = torch.tensor([t - 1, b1 ** (t - 1), b2 ** (t - 1), 0.0], dtype=torch.float64, device="cuda")
    got = p.cuda()
    optim.adamw_step([got], [torch.zeros(n, device="cuda")], [qm], [qv], count, scales=[s], lr=lr, betas=(b1, b2), eps=0.0,
                     weight_decay=0.0)
    step = lr * (b1 * M / (1 - b1 ** t)) / (b2 * V / (1 - b2 ** t)).sqrt()
    # four roundings each in reading m and v, two in each moment's update, a root, a quotient and three factors
    allowed = 2.0 ** -24 * (16 * step.abs() + 4 * p.double().abs())
    assert ((got.cpu().double() - (p.double() - step)).abs() <= allowed).all()


def test_a_max_norm_that_float32_does_not_have(optim):
    """One that would round to zero is refused, as zero is; the least one clips to almost nothing."""
    p, g = torch.zeros(4, device="cuda"), torch.ones(4, device="cuda")
    m, v, _ = optim.empty_moments(p)
    step = lambda most: optim.adamw_step([p], [g], [m], [v], optim.counter(), max_norm=most, **HYPER)  # noqa: E731
    with pytest.raises(AssertionError, match="max_norm"):
        step(1e-46)
    assert not m.any()
    assert float(step(1e-30)) == 2.0
    assert ((m > 0) & (m < 1e-30)).all()


def test_a_parameter_without_a_gradient_is_left_alone(optim):
    """Nothing of it is written, and what autograd has saved of it stays good."""
    p, q = torch.ones(4, device="cuda"), torch.full((4,), 2.0, device="cuda")
    M = [optim.empty_moments(t) for t in (p, q)]
    copies = [torch.zeros(4, device="cuda"), torch.zeros(4, device="cuda")]
    x = torch.ones(4, device="cuda", requires_grad=True)
    y = (x * q).sum()                                                # (saves q)
    lists = [p, *M[0][:2], copies[0]], [q, *M[1][:2], copies[1]]
    before = [[t._version for t in ts] for ts in lists]
    optim.adamw_step([p, q], [torch.ones_like(p), None], [m for m, _, _ in M], [v for _, v, _ in M], optim.counter(),
                     copies=copies, **HYPER)
    assert all(t._version > b for t, b in zip(lists[0], before[0]))
    assert [t._version for t in lists[1]] == before[1] and not copies[1].any()
    y.backward()
    assert torch.equal(x.grad, q)
