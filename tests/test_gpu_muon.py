"""The Muon step and its orthogonalised updates against the formula in 64 bits."""
import copy
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
A, B, C = 3.4445, -4.7750, 2.0315


@pytest.fixture(scope="module")
def optim():
    import paralleltnnlayers_amd as cp4
    from paralleltnnlayers_amd import optim
    cp4.lib()
    return optim


def polar(u, steps=5, eps=1e-7):
    """The formula in 64 bits, of a matrix or a stack of them."""
    u = u.double().cpu()
    x = u / (u.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.mT
    for _ in range(steps):
        s = x @ x.mT
        x = A * x + (B * s + C * (s @ s)) @ x
    return x.mT if tall else x


def matrix(*shape, seed=0, dtype=torch.float32, spread=0.0):
    """Noise, with ``spread`` > 0 a few directions of up to 10^spread times its size on top."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g)
    if spread:
        k = min(8, shape[-1], shape[-2])
        x = x + (torch.randn(*shape[:-1], k, generator=g) * 10 ** torch.linspace(spread, 0, k)) @ torch.randn(*shape[:-2], k, shape[-1], generator=g)
    return (x * 1e-3).to(dtype).cuda()


def off(got, want):
    got, want = got.double().cpu(), want.double()
    return float((got - want).norm() / want.norm())


def allowed(dtype, steps=5):
    """What an output's norm may be off by, relative: its own rounding (uniform up to half a step: a root of 3 smaller in
    the norm, a quarter of margin), and of the iteration: X's and A's roundings of 2^-23 and fp32 sums, which each step
    multiplies by up to 3.4445 in the directions that are still small while the others stay: 3.4445^4 = 141 of them at the end
    at most, 2^-23 each and some three a step."""
    return torch.finfo(dtype).eps / 2 * 0.75 + 3 * 141 * 2.0 ** -23


SHAPES = [(1, 1), (1, 64), (64, 1), (3, 16), (7, 1001), (777, 7), (16, 16), (17, 300), (300, 17), (32, 512), (33, 40), (48, 200),
          (64, 64), (64, 1000), (1000, 64), (65, 65), (65, 2000), (2000, 65), (96, 128), (128, 128), (129, 257), (200, 100),
          (256, 256), (333, 1001), (1000, 777), (512, 2048)]


@pytest.mark.parametrize("dtype", list(DTYPES), ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_orthogonalize(optim, shape, dtype):
    u = matrix(*shape, dtype=DTYPES[dtype], spread=0.5 if shape[0] % 2 else 0.0)
    x = optim.orthogonalize(u)
    assert x.dtype == u.dtype and x.shape == u.shape
    assert off(x, polar(u)) <= allowed(u.dtype)


def test_large_launches(optim):
    """Enough tiles for the large shape of them, in one launch of several entries, and the two depths of a matrix with a long side."""
    us = [matrix(1024, 1536, seed=1), matrix(1536, 1024, seed=2), matrix(2, 640, 700, seed=3), matrix(100, 9000, seed=4), matrix(2500, 2100, seed=5)]
    for u, x in zip(us, optim.orthogonalize(us)):
        assert off(x, polar(u)) <= allowed(u.dtype)


def test_small_singular_values_count(optim):
    """A direction a thousand times smaller than the largest comes out as the polynomial takes it, not as noise."""
    for shape in ((16, 400), (64, 300), (96, 400)):
        q, _ = torch.linalg.qr(torch.randn(shape[0], shape[0], dtype=torch.float64, generator=torch.Generator().manual_seed(1)))
        r, _ = torch.linalg.qr(torch.randn(shape[1], shape[0], dtype=torch.float64, generator=torch.Generator().manual_seed(2)))
        s = torch.ones(shape[0], dtype=torch.float64)
        s[-1] = 1e-3
        u = ((q * s) @ r.T).float().cuda()
        x = optim.orthogonalize(u).double().cpu()
        along = float(q[:, -1] @ x @ r[:, -1])
        want = float(q[:, -1] @ polar(u) @ r[:, -1])
        assert abs(along - want) <= 2e-3 * abs(want)                 # (u's own rounding is 1e-3 / 2^24 / 1e-3 and is in both)


@pytest.mark.parametrize("steps", [1, 2, 3, 16])
@pytest.mark.parametrize("shape", [(20, 50), (90, 70)], ids=str)
def test_steps(optim, shape, steps):
    u = matrix(*shape)
    # (past five steps the polynomial's slope is below 2 where the values are, on the mean below 1.3, and errors grow slowly)
    assert off(optim.orthogonalize(u, steps=steps), polar(u, steps)) <= allowed(u.dtype) * (1 if steps < 16 else 20)


def test_stacks_are_orthogonalised_one_by_one(optim):
    for shape in ((5, 7, 64, 9), (3, 100, 80)):
        u = matrix(*shape)
        x = optim.orthogonalize(u)
        flat = u.view(-1, *shape[-2:])
        alone = torch.stack([optim.orthogonalize(m) for m in flat]).view(shape)
        assert off(x, alone.cpu()) <= 1e-6 and off(x, polar(u)) <= allowed(u.dtype)


def test_scale_zero_and_strides(optim):
    for shape in ((12, 100), (100, 130)):
        u = matrix(*shape)
        want = optim.orthogonalize(u, eps=1e-30)
        # eps is 3e-29 of u's norm, half a step of fp64 2^-53 = 1e-16: at 2^100 times that the sums are the same but for their
        # exponent.  At 2^-60 times it, 3e-11 of the norm, they are not, and every rounding behind may fall the other way:
        # both results are as far off the formula's as they may be.
        assert torch.equal(optim.orthogonalize(u * 2.0 ** 100, eps=1e-30), want)
        assert off(optim.orthogonalize(u * 2.0 ** -60, eps=1e-30), want.cpu()) <= 2 * allowed(u.dtype)
        assert not optim.orthogonalize(torch.zeros_like(u)).any()
        wide = torch.zeros(shape[0], shape[1] + 3, device="cuda")
        wide[:, 1:-2] = u
        assert torch.equal(optim.orthogonalize(wide[:, 1:-2], eps=1e-30), want)
        odd = torch.zeros(u.numel() + 1, device="cuda")[1:].view(shape)
        out = torch.zeros(u.numel() + 1, dtype=torch.bfloat16, device="cuda")[1:].view(shape)
        assert optim.orthogonalize(odd.copy_(u), eps=1e-30, out=out) is out and torch.equal(out, want.bfloat16())
    assert optim.orthogonalize(torch.zeros(0, 4, 5, device="cuda")).shape == (0, 4, 5)
    assert optim.orthogonalize([]) == []


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_what_is_not_finite_stays_with_its_matrix(optim, bad):
    us = [matrix(9, 40), matrix(70, 90), matrix(9, 40, seed=1), matrix(70, 90, seed=1), matrix(3, 70, 66, seed=1)]
    want = optim.orthogonalize(us)
    us[0][3, 3] = us[1][5, 5] = us[4][1, 0, 0] = bad
    got = optim.orthogonalize(us)
    assert got[0].isnan().all() and got[1].isnan().all() and got[4][1].isnan().all()
    assert torch.equal(got[2], want[2]) and torch.equal(got[3], want[3])
    assert torch.equal(got[4][0], want[4][0]) and torch.equal(got[4][2], want[4][2])


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("types", [("f32", "f32", None), ("f32", "bf16", "bf16"), ("f32", "f16", "f16"), ("bf16", "bf16", None), ("f16", "f32", None)],
                         ids=lambda t: "-".join(map(str, t)))
def test_step(optim, types, nesterov):
    param, grad, copied = (t and DTYPES[t] for t in types)
    shapes = [(13, 500), (500, 13), (4, 8, 100), (64, 3), (130, 200), (200, 130), (2, 70, 70)]
    ps = [(20 * matrix(*s, seed=i)).to(param) for i, s in enumerate(shapes)]
    ms = [matrix(*s, seed=50 + i, spread=0.3) for i, s in enumerate(shapes)]
    gs = [matrix(*s, seed=100 + i).to(grad) for i, s in enumerate(shapes)]
    cs = [torch.zeros_like(p, dtype=copied) for p in ps] if copied else None
    before = [t.clone() for t in ps], [t.clone() for t in ms]
    versions = [t._version for t in ps + ms]
    gs[1] = None                                                     # (left alone)
    optim.muon_step(ps, gs, ms, lr=0.1, momentum=0.9, nesterov=nesterov, weight_decay=0.2, copies=cs)
    assert torch.equal(ps[1], before[0][1]) and torch.equal(ms[1], before[1][1])
    assert [t._version - v for t, v in zip(ps + ms, versions)] == [0 if i % 7 == 1 else 1 for i in range(14)]
    for i, g in enumerate(gs):
        if g is None:
            continue
        g = g.double().cpu()
        m = before[1][i].double().cpu() * 0.9 + g
        u = g + 0.9 * m if nesterov else m
        # two roundings of an fp32 m; the orthogonalised matrix's error times the rate, and p's own roundings
        assert off(ms[i], m) <= 2.0 ** -23
        rate = 0.1 * math.sqrt(max(1.0, u.shape[-2] / u.shape[-1]))
        x = polar(u)
        p = before[0][i].double().cpu() * (1 - 0.1 * 0.2) - rate * x
        bound = float(p.norm()) * (torch.finfo(param).eps / 2 + 3 * 2.0 ** -24) + rate * float(x.norm()) * allowed(torch.float32)
        assert float((ps[i].double().cpu() - p).norm()) <= bound
        if copied:
            assert torch.equal(cs[i], ps[i].to(copied))


def test_repeats_and_graph(optim):
    ps = [matrix(16, 300), matrix(160, 300), matrix(3, 300, 40)]
    gs = [matrix(*p.shape, seed=5) for p in ps]
    ms = [torch.zeros_like(p) for p in ps]
    start = [t.clone() for t in ps]
    side = torch.cuda.Stream()
    optim.muon_step([p.clone() for p in ps], gs, [m.clone() for m in ms], lr=0.1)     # (outside the capture)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        optim.muon_step(ps, gs, ms, lr=0.1)
    eager_p, eager_m = [t.clone() for t in start], [torch.zeros_like(t) for t in ps]
    for k in range(4):
        for g in gs:
            g.mul_(1.5)
        graph.replay()
        side.wait_stream(torch.cuda.current_stream())
        optim.muon_step(eager_p, gs, eager_m, lr=0.1, stream=side)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(ps + ms, eager_p + eager_m)), k


def test_optimizer(optim):
    torch.manual_seed(0)
    make = lambda: [torch.nn.Parameter(matrix(20, 64)), torch.nn.Parameter(matrix(2, 96, 70).bfloat16())]  # noqa: E731
    ps, lists = make(), make()
    opt = optim.Muon([{"params": [ps[0]], "lr": 0.3}, {"params": [ps[1]], "nesterov": False}], lr=0.1, weight_decay=0.1)
    master, ms = lists[1].detach().float(), [torch.zeros(20, 64, device="cuda"), torch.zeros(2, 96, 70, device="cuda")]
    for k in range(3):
        for i, p in enumerate(ps):
            p.grad = matrix(*p.shape, seed=10 * k + i).to(p.dtype)
        opt.step()
        optim.muon_step([lists[0].data], [ps[0].grad], ms[:1], lr=0.3, weight_decay=0.1)
        optim.muon_step([master], [ps[1].grad], ms[1:], lr=0.1, weight_decay=0.1, nesterov=False, copies=[lists[1].data])
        assert all(torch.equal(a, b) for a, b in zip(ps, lists))
        if k == 1:                                                   # goes on from a saved state, and from a copy
            saved = copy.deepcopy(opt.state_dict())
            fresh = optim.Muon([{"params": [ps[0]], "lr": 0.3}, {"params": [ps[1]], "nesterov": False}], lr=0.1, weight_decay=0.1)
            fresh.load_state_dict(saved)
            opt = fresh
            assert all(s["momentum_buffer"].dtype == torch.float32 for s in opt.state.values())
    again = copy.deepcopy(opt)
    assert again.masters is True
    ps[0].grad = None
    before = ps[0].detach().clone()
    opt.step()
    assert torch.equal(ps[0], before)


def test_refusals(optim):
    from paralleltnnlayers_amd import Cp4Error
    p, g, m = matrix(8, 16), matrix(8, 16, seed=1), torch.zeros(8, 16, device="cuda")
    for call in (lambda: optim.muon_step([p], [g.cpu()], [m], lr=0.1), lambda: optim.muon_step([p], [g], [m.half()], lr=0.1),
                 lambda: optim.muon_step([p], [g[:4]], [m], lr=0.1), lambda: optim.muon_step([p, p], [g], [m], lr=0.1),
                 lambda: optim.muon_step([p.t()], [g.t()], [m.t()], lr=0.1), lambda: optim.muon_step([p[0]], [g[0]], [m[0]], lr=0.1),
                 lambda: optim.muon_step([p], [g.double()], [m], lr=0.1), lambda: optim.muon_step([p], [g], [m], lr=0.1, steps=0),
                 lambda: optim.muon_step([p], [g], [m], lr=0.1, steps=17), lambda: optim.orthogonalize(torch.zeros(2, 70000, device="cuda")),
                 lambda: optim.orthogonalize(g, out=torch.zeros(16, 8, device="cuda"))):
        with pytest.raises(AssertionError):
            call()
    for kw in (dict(lr=-1.0), dict(lr=math.nan), dict(lr=0.1, momentum=1.0), dict(lr=0.1, weight_decay=-1.0), dict(lr=0.1, eps=0.0)):
        with pytest.raises(Cp4Error):
            optim.muon_step([p], [g], [m], **kw)
    with pytest.raises(ValueError, match="two dimensions"):
        optim.Muon([torch.nn.Parameter(torch.zeros(3, device="cuda"))])
    for kw in (dict(lr=-1), dict(momentum=1.0), dict(steps=0), dict(eps=0.0)):
        with pytest.raises(ValueError):
            optim.Muon([torch.nn.Parameter(p.clone())], **kw)
    assert torch.equal(p, matrix(8, 16))
    flat = torch.zeros(200, device="cuda")
    for call in (lambda: optim.muon_step([p, p], [g, g], [m, torch.zeros_like(m)], lr=0.1),              # the same one twice
                 lambda: optim.muon_step([p, matrix(8, 16)], [g, g], [m, m], lr=0.1), lambda: optim.muon_step([p], [g], [g], lr=0.1),
                 lambda: optim.muon_step([p], [p], [m], lr=0.1), lambda: optim.muon_step([p], [g], [m], lr=0.1, copies=[p]),
                 lambda: optim.orthogonalize([g], out=[g.view(-1)[:0].view(0, 16)]),
                 lambda: optim.orthogonalize(flat[:128].view(8, 16), out=flat[8:136].view(8, 16)),
                 lambda: optim.orthogonalize([g, matrix(8, 16)], out=[m, g])):
        with pytest.raises(AssertionError):
            call()
    assert torch.equal(p, matrix(8, 16)) and torch.equal(g, matrix(8, 16, seed=1)) and not m.any()


@pytest.mark.parametrize("shape", [(12, 700), (700, 12), (50, 90), (100, 300), (300, 100)], ids=str)
def test_in_its_own_place(optim, shape):
    for dtype in DTYPES.values():
        u = matrix(3, *shape, dtype=dtype)
        want = optim.orthogonalize(u)
        assert optim.orthogonalize(u, out=u) is u and torch.equal(u, want)


def test_many_small_matrices(optim):
    """More than one launch takes (each has up to 65536 tiles of its long sides)."""
    u = torch.randn(70000, 2, 3, generator=torch.Generator().manual_seed(1)).cuda()
    x = optim.orthogonalize(u)
    assert off(x, polar(u)) <= allowed(u.dtype)
    assert torch.equal(optim.orthogonalize(u[65000:].clone()), x[65000:])


@pytest.mark.parametrize("shape", [(520, 64, 65536), (260, 65, 65536)], ids=str)
def test_stacks_beyond_32_bit_offsets(optim, shape):
    u = torch.zeros(shape, device="cuda")
    assert u.numel() * 4 > 1 << 32
    last = matrix(*shape[1:], seed=3)
    u[-1] = last
    u[0] = matrix(*shape[1:], seed=4)
    x = optim.orthogonalize(u, out=u)
    assert x is u and not u[1:-1].any()
    assert off(u[-1], polar(last)) <= allowed(u.dtype)
