"""The AdamW step over many tensors: against the formula in 64 bits, and bit by bit against its
fp32 operations one after the other (numpy), codes and scales of 8-bit moments included."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
F = np.float32
HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.02)
# below, at and beyond a lane's four values, a block, a wave's turn
SIZES = (1, 3, 4, 5, 63, 255, 256, 257, 511, 1000, 1023, 1024, 1025, 4099, 70001)


@pytest.fixture(scope="module")
def optim():
    from paralleltnnlayers_amd import capi, optim
    capi.lib()
    return optim


def gradients(gen, n, std=1e-2):
    size = torch.exp(2 * torch.randn(n, generator=gen))           # magnitudes over several powers of ten
    return torch.randn(n, generator=gen) * size * std


def codes(m, v):
    """(q of m, q of v, scales) of float32 moments, 256 at a time."""
    n = len(m)
    pad = lambda t: np.concatenate([t, np.zeros(-n % 256, F)]).reshape(-1, 256)
    m, v = pad(m), pad(v)
    tops = np.stack([np.abs(m).max(1), v.max(1)])
    tops[tops < 2.0 ** -126] = 0
    with np.errstate(divide="ignore"):
        over = np.where(tops > 0, F(1) / tops, F(0)).astype(F)[:, :, None]
    qm = np.rint(np.sqrt(np.abs(m) * over[0]) * F(127)) * np.sign(m)
    qv = np.rint(np.sqrt(np.sqrt(v * over[1])) * F(255))
    qv[(qv < 1) & (v > 0) & (over[1] > 0)] = 1
    return qm.ravel()[:n].astype(np.int8), qv.ravel()[:n].astype(np.uint8), tops.astype(F)


def values(qm, qv, tops):
    at = np.arange(len(qm)) // 256
    m, v = qm.astype(F), qv.astype(F)
    v2 = v * v
    return np.abs(m) * m * (tops[0] * F(1 / 127 ** 2))[at], v2 * v2 * (tops[1] * F(1 / 255 ** 4))[at]


def numpy_step(p, g, m, v, t, lr, betas, eps, weight_decay, factor=F(1)):
    """One step in float32, operation by operation; t: steps including this one."""
    b1, b2 = betas
    p1 = p2 = 1.0
    for _ in range(t):
        p1, p2 = p1 * b1, p2 * b2
    rate, root = F(lr / (1 - p1)), F(1 / np.sqrt(1 - p2))
    g = g * factor
    m = m * F(b1) + g * F(1 - b1)
    v = v * F(b2) + (g * g) * F(1 - b2)
    p = p * F(1 - lr * weight_decay) - (m / (np.sqrt(v) * root + F(eps))) * rate
    return p, m, v


def narrow(p, dtype):
    return torch.from_numpy(p.copy()).to(DTYPES[dtype])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("grad", list(DTYPES))
@pytest.mark.parametrize("param", list(DTYPES))
def test_bit_by_bit(optim, param, grad, bits):
    """Three steps over tensors of all sizes."""
    gen = torch.Generator().manual_seed(1)
    P = [(torch.randn(n, generator=gen) * 0.1).to(DTYPES[param]) for n in SIZES]
    state = [[np.zeros(n, F), np.zeros(n, F)] for n in SIZES]
    params = [p.cuda() for p in P]
    moments = [optim.empty_moments(p, bits) for p in params]
    count = optim.counter()
    for t in (1, 2, 3):
        G = [gradients(gen, n).to(DTYPES[grad]) for n in SIZES]
        optim.adamw_step(params, [g.cuda() for g in G], [m for m, _, _ in moments], [v for _, v, _ in moments],
                         count, scales=[s for _, _, s in moments], **HYPER)
        for i, n in enumerate(SIZES):
            p, m, v = numpy_step(P[i].float().numpy(), G[i].float().numpy(), *state[i], t, **HYPER)
            P[i] = narrow(p, param)
            assert torch.equal(params[i].cpu(), P[i]), f"step {t}, {n} values: parameters"
            if bits == 32:
                state[i] = [m, v]
                got = [moments[i][0].cpu().numpy(), moments[i][1].cpu().numpy()]
                assert all(np.array_equal(a, b) for a, b in zip(got, state[i])), f"step {t}, {n} values: moments"
            else:
                q = codes(m, v)
                got = [x.cpu().numpy() for x in moments[i]]
                assert all(np.array_equal(a, b) for a, b in zip(got, q)), f"step {t}, {n} values: codes"
                state[i] = list(values(*q))
    assert count.cpu()[0] == 3 and count.cpu()[3] == 0


def test_against_64_bits(optim):
    """Five steps; each rounds a value six times or so, and m and v remember the last ten or hundred."""
    gen = torch.Generator().manual_seed(2)
    n = 5000
    p = torch.randn(n, generator=gen) * 0.1
    P, M, V = p.double(), torch.zeros(n).double(), torch.zeros(n).double()
    param, count = p.cuda(), optim.counter()
    m, v, _ = optim.empty_moments(param)
    moved = torch.zeros(n).double()
    for t in range(1, 6):
        g = gradients(gen, n)
        optim.adamw_step([param], [g.cuda()], [m], [v], count, **HYPER)
        G = g.double()
        M, V = 0.9 * M + 0.1 * G, 0.99 * V + 0.01 * G * G
        step = HYPER["lr"] * (M / (1 - 0.9 ** t)) / ((V / (1 - 0.99 ** t)).sqrt() + HYPER["eps"])
        P = P * (1 - HYPER["lr"] * HYPER["weight_decay"]) - step
        moved += step.abs()
    # a step's numerator may cancel: its error is that of the sizes that it is a sum of
    size = 0.1 * sum(0.9 ** (5 - t) for t in range(1, 6)) * HYPER["lr"] * 5
    allowed = 2.0 ** -24 * (5 * 2 * P.abs() + 16 * (moved + size) * 30)
    assert ((param.cpu().double() - P).abs() <= allowed).all()
    assert ((v.cpu().double() - V).abs() <= 2.0 ** -24 * 20 * V).all()


@pytest.mark.parametrize("copy", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("bits", [32, 8])
def test_copies(optim, bits, copy):
    gen = torch.Generator().manual_seed(3)
    P = [torch.randn(n, generator=gen).cuda() for n in SIZES]
    C = [torch.zeros(n, dtype=DTYPES[copy], device="cuda") for n in SIZES]
    G = [gradients(gen, n).cuda() for n in SIZES]
    M = [optim.empty_moments(p, bits) for p in P]
    lists = [[m for m, _, _ in M], [v for _, v, _ in M]]
    some = [c if i % 3 else None for i, c in enumerate(C)]           # (not every parameter has one)
    optim.adamw_step(P, G, *lists, optim.counter(), scales=[s for _, _, s in M], copies=some, **HYPER)
    for i, (p, c) in enumerate(zip(P, C)):
        assert torch.equal(c, p.to(c.dtype)) if i % 3 else not c.any()


@pytest.mark.parametrize("bits", [32, 8])
def test_tensors_that_start_anywhere(optim, bits):
    """Views that start off every vector's boundary give the same bits."""
    gen = torch.Generator().manual_seed(4)
    n = 3001
    p, g = torch.randn(n, generator=gen).cuda(), gradients(gen, n).cuda()

    def run(off):
        put = lambda t: torch.cat([t.new_zeros(off), t.flatten()])[off:]
        q, grad, c = put(p), put(g.bfloat16()), put(torch.zeros(n, dtype=torch.float16, device="cuda"))
        m, v, s = optim.empty_moments(q, bits)
        m, v = put(m), put(v)
        if s is not None:
            s = torch.cat([s.new_zeros(2, off), s], 1)[:, off:]
        for _ in range(2):
            optim.adamw_step([q], [grad], [m], [v], count, scales=None if s is None else [s], copies=[c], **HYPER)
        return [t.clone() for t in (q, m, v, c)] + ([] if s is None else [s.clone()])

    count = optim.counter()
    want = run(0)
    for off in (1, 2, 3, 5):
        count = optim.counter()
        assert all(torch.equal(a, b) for a, b in zip(run(off), want)), off


def test_many_tensors(optim):
    """More than one launch holds, gradients that are not there, tensors without values."""
    gen = torch.Generator().manual_seed(5)
    sizes = [1 + 37 * i % 700 for i in range(450)]
    sizes[7] = sizes[200] = 0
    P = [torch.randn(n, generator=gen) for n in sizes]
    G = [gradients(gen, n) for n in sizes]
    params = [p.cuda() for p in P]
    bits = [8 if i % 3 == 0 else 32 for i in range(len(sizes))]
    M = [optim.empty_moments(p, b) for p, b in zip(params, bits)]
    count = optim.counter()
    optim.adamw_step(params, [None if i % 5 == 0 else g.cuda() for i, g in enumerate(G)], [m for m, _, _ in M],
                     [v for _, v, _ in M], count, scales=[s for _, _, s in M], **HYPER)
    for i, n in enumerate(sizes):
        want = P[i].numpy()
        if i % 5:
            want = numpy_step(want, G[i].numpy(), np.zeros(n, F), np.zeros(n, F), 1, **HYPER)[0]
        assert np.array_equal(params[i].cpu().numpy(), want), i
    assert count.cpu()[0] == 1


def test_clipping(optim):
    """The norm of all gradients, of mixed types, and the step that it leads to."""
    gen = torch.Generator().manual_seed(6)
    sizes = list(SIZES) * 20                                         # (more than a launch of the norm takes)
    kinds = [list(DTYPES)[i % 3] for i in range(len(sizes))]
    P = [torch.randn(n, generator=gen) for n in sizes]
    G = [gradients(gen, n).to(DTYPES[k]) for n, k in zip(sizes, kinds)]
    total = float(torch.cat([g.double() for g in G]).norm())
    for scale in (1.0, 0.125):
        for most in (0.5 * total * scale, 2 * total * scale):
            params = [p.cuda() for p in P]
            M = [optim.empty_moments(p) for p in params]
            norm = optim.adamw_step(params, [g.cuda() for g in G], [m for m, _, _ in M], [v for _, v, _ in M],
                                    optim.counter(), max_norm=most, grad_scale=scale, **HYPER)
            # a sum in 64 bits, rounded once
            assert abs(float(norm) - total * scale) <= 2.0 ** -23 * total * scale
            factor = F(scale) * min(F(most) / (F(norm.cpu().numpy()) + F(1e-6)), F(1))
            for i in range(0, len(sizes), 17):
                want = numpy_step(P[i].numpy(), G[i].float().numpy(), np.zeros(sizes[i], F), np.zeros(sizes[i], F),
                                  1, factor=factor, **HYPER)
                assert np.array_equal(params[i].cpu().numpy(), want[0]), (scale, most, i)


@pytest.mark.parametrize("spoiled", [float("inf"), float("nan")])
@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_that_is_skipped(optim, bits, spoiled):
    gen = torch.Generator().manual_seed(7)
    P = [torch.randn(n, generator=gen).cuda() for n in (300, 5000)]
    G = [gradients(gen, n).cuda() for n in (300, 5000)]
    M = [optim.empty_moments(p, bits) for p in P]
    count = optim.counter()
    step = lambda: optim.adamw_step(P, G, [m for m, _, _ in M], [v for _, v, _ in M], count,
                                    scales=[s for _, _, s in M], max_norm=1.0, **HYPER)
    state = lambda: [t.clone() for t in P + [x for three in M for x in three if x is not None] + [count]]
    step()
    before = state()
    good = G[1][4321].clone()
    G[1][4321] = spoiled
    assert not torch.isfinite(step())
    assert all(torch.equal(a, b) for a, b in zip(state(), before))
    G[1][4321] = good
    step()
    assert count.cpu()[0] == 2 and not torch.equal(P[0], before[0])


def test_spoiled_gradients_without_clipping(optim):
    """32 bits: the value alone; 8 bits: its block of 256, loudly."""
    gen = torch.Generator().manual_seed(8)
    n = 1000
    p, g = torch.randn(n, generator=gen), gradients(gen, n)
    g[300] = float("nan")
    for bits in (32, 8):
        q = p.cuda()
        m, v, s = optim.empty_moments(q, bits)
        count = optim.counter()
        step = lambda: optim.adamw_step([q], [g.cuda()], [m], [v], count, scales=[s], **HYPER)
        step()
        assert q.isnan().nonzero().flatten().tolist() == [300]
        if bits == 8:
            assert s.isnan().cpu().tolist() == [[False, True, False, False]] * 2
            a, b = optim.moment_values([m], [v], [s])
            for t in (a[0], b[0]):
                assert t[256:512].isnan().all() and not t[:256].isnan().any() and not t[512:].isnan().any()
        else:
            assert m.isnan().nonzero().flatten().tolist() == [300]


def test_tiny_and_zero_moments(optim):
    """A second moment above zero keeps a code; blocks of nothing, and of less than the smallest normal number."""
    v = torch.zeros(1024)
    v[0], v[1] = 1.0, 1e-30                       # far below the smallest level of its block
    v[512], v[513] = 1e-40, 1e-41                 # a block of denormal numbers
    m = torch.zeros(1024)
    m[0], m[1], m[2] = -1.0, 1e-9, -0.3
    qm, qv, s = optim.empty_moments(torch.empty(1024, device="cuda"), 8)
    optim.set_moments([qm], [qv], [s], ([m.cuda()], [v.cuda()]))
    want = codes(m.numpy(), v.numpy())
    assert all(np.array_equal(a.cpu().numpy(), b) for a, b in zip((qm, qv, s), want))
    assert qv[1] == 1 and qv[2] == 0 and not s[:, 1:].any()
    a, b = optim.moment_values([qm], [qv], [s])
    assert a[0][0] == -1.0 and a[0][1] == 0 and abs(float(a[0][2]) + 0.3) < 0.3 * 2 / 127 / 0.5
    assert 0 < float(b[0][1]) < 1e-9 and float(b[0][0]) == pytest.approx(1.0, rel=2.0 ** -22)


def test_levels_are_their_own_codes(optim):
    """Every level of a block comes back as itself."""
    q = torch.arange(256)
    top = torch.tensor([3.7e-3, 2.2e-5])
    qm = torch.cat([(q - 127).clamp(max=127)]).to(torch.int8)
    m, v = values(qm.numpy(), q.to(torch.uint8).numpy(), top[:, None].numpy())
    m8, v8, s = optim.empty_moments(torch.empty(256, device="cuda"), 8)
    optim.set_moments([m8], [v8], [s], ([torch.from_numpy(m).cuda()], [torch.from_numpy(v).cuda()]))
    assert torch.equal(m8.cpu(), qm) and torch.equal(v8.cpu(), q.to(torch.uint8))


def test_recorded_in_a_graph(optim):
    """The count of steps is the device's: replays are the steps 2, 3, ..."""
    gen = torch.Generator().manual_seed(9)
    P0 = [torch.randn(n, generator=gen).cuda() for n in (700, 3000)]
    G = [gradients(gen, n).cuda() for n in (700, 3000)]

    def program():
        P = [p.clone() for p in P0]
        M = [optim.empty_moments(p, b) for p, b in zip(P, (32, 8))]
        count = optim.counter()
        run = lambda: optim.adamw_step(P, G, [m for m, _, _ in M], [v for _, v, _ in M], count,
                                       scales=[s for _, _, s in M], max_norm=0.5, **HYPER)
        return P, count, run

    P, count, run = program()
    Q, other, eager = program()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = run()
    eager()
    for i in range(4):
        for g in G:
            g.mul_(1.5)
        graph.replay()
        torch.cuda.synchronize()
        want = eager()
        assert torch.equal(norm, want) and torch.equal(count, other)
        assert all(torch.equal(a, b) for a, b in zip(P, Q)), i


def test_another_stream(optim):
    gen = torch.Generator().manual_seed(10)
    p, g = torch.randn(4000, generator=gen).cuda(), gradients(gen, 4000).cuda()
    q = p.clone()
    a, b = optim.empty_moments(p)[:2], optim.empty_moments(q)[:2]
    n1 = optim.adamw_step([p], [g], [a[0]], [a[1]], optim.counter(), max_norm=1.0, **HYPER)
    count = optim.counter()
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    n2 = optim.adamw_step([q], [g], [b[0]], [b[1]], count, max_norm=1.0, stream=st, **HYPER)
    st.synchronize()
    assert torch.equal(p, q) and torch.equal(n1, n2)


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer(optim, bits):
    """The optimizer: groups with rates of their own, masters, state to and from a checkpoint."""
    def program():
        torch.manual_seed(11)
        big = torch.nn.Parameter(torch.randn(80, 90, device="cuda").bfloat16())
        small = torch.nn.Parameter(torch.randn(33, device="cuda"))
        idle = torch.nn.Parameter(torch.randn(5, device="cuda"))
        opt = optim.AdamW([dict(params=[big, idle]), dict(params=[small], lr=1e-2, weight_decay=0.0)], lr=1e-3,
                          state_bits=bits, max_norm=1.0)
        return opt, big, small, idle

    def feed(t, *params):
        gen = torch.Generator().manual_seed(100 + t)
        for p in params:
            p.grad = torch.randn(p.shape, generator=gen).to(p.dtype).cuda()

    opt, big, small, idle = program()
    still = idle.detach().clone()
    seen = big._version
    for t in range(3):
        feed(t, big, small)
        opt.step()
    assert big._version > seen
    assert torch.equal(idle, still) and idle not in opt.state
    master = opt.state[big]["master"]
    assert master.dtype == torch.float32 and torch.equal(big, master.bfloat16())
    assert opt.state[big]["exp_avg"].dtype == (torch.int8 if bits == 8 else torch.float32)
    assert opt.state[small]["exp_avg"].dtype == torch.float32
    assert float(opt.last_norm) > 1.0
    # the lists' step does the same
    want, norm = program(), None
    gs = []
    lists = {k: optim.empty_moments(p, b) for k, p, b in (("b", want[1], bits), ("s", want[2], 32))}
    m32, p32, counters = want[1].detach().float(), want[2].detach().clone(), [optim.counter(), optim.counter()]
    from paralleltnnlayers_amd import capi
    for t in range(3):
        feed(t, want[1], want[2])
        norm = capi._native.adamw_step(
            [m32, p32], [want[1].grad, want[2].grad], [lists["b"][0], lists["s"][0]], [lists["b"][1], lists["s"][1]],
            [lists["b"][2], None], None, [0, 1],
            [(1e-3, 0.9, 0.999, 1e-8, 0.01, counters[0]), (1e-2, 0.9, 0.999, 1e-8, 0.0, counters[1])], 1.0, 1.0, None)
    assert torch.equal(m32, master) and torch.equal(p32, small.detach()) and torch.equal(norm, opt.last_norm)
    # a checkpoint
    saved = {k: p.detach().clone() for k, p in (("big", big), ("small", small))}
    state = opt.state_dict()
    import copy
    state = copy.deepcopy(state)
    feed(7, big, small)
    opt.step()
    new, big2, small2, _ = program()
    with torch.no_grad():
        big2.copy_(saved["big"])
        small2.copy_(saved["small"])
    new.load_state_dict(state)
    assert new.state[big2]["master"].dtype == torch.float32
    feed(7, big2, small2)
    new.step()
    assert torch.equal(big2, big) and torch.equal(small2, small)
    assert torch.equal(new.state[big2]["exp_avg"], opt.state[big]["exp_avg"])


def test_optimizer_trains(optim):
    """Layers of the library under this optimizer and under torch's: the same losses.  The steps' roundings,
    some 2^-22 of a parameter's change each, reach the loss with about its own relative size."""
    from paralleltnnlayers_amd import torch_ops

    def losses(make):
        torch.manual_seed(12)
        conv = torch_ops.CP4Conv2d(8, 16, 3, 4, bias=True, activation="relu")
        head = torch_ops.AdapterLinear(16, 10, rank=4, adapters=2)
        opt = make([*conv.parameters(), *head.parameters()])
        x, ids = torch.randn(32, 8, 12, 12, device="cuda"), torch.arange(32, device="cuda").remainder(2).int()
        label = torch.randint(0, 10, (32,), device="cuda")
        seen = []
        for _ in range(10):
            opt.zero_grad()
            loss = torch.nn.functional.cross_entropy(head(conv(x).mean((2, 3)), ids), label)
            loss.backward()
            opt.step()
            seen.append(float(loss))
        return seen

    ours = losses(lambda p: optim.AdamW(p, lr=1e-2))
    theirs = losses(lambda p: torch.optim.AdamW(p, lr=1e-2, weight_decay=0.01))
    assert ours[-1] < ours[0]
    assert ours == pytest.approx(theirs, rel=1e-3)


def test_refusals(optim):
    from paralleltnnlayers_amd import capi
    p, g = torch.zeros(600, device="cuda"), torch.zeros(600, device="cuda")
    m, v, _ = optim.empty_moments(p)
    m8, v8, s8 = optim.empty_moments(p, 8)
    c = optim.counter()
    ok = dict(params=[p], grads=[g], exp_avgs=[m], exp_avg_sqs=[v], counter=c, lr=1e-3)
    step = lambda **kw: optim.adamw_step(**{**ok, **kw})
    bad = [
        dict(grads=[]), dict(grads=[g[:599]]), dict(grads=[g.cpu()]), dict(grads=[g.double()]), dict(params=[p.cpu()]),
        dict(params=[p[::2]], grads=[g[::2]]), dict(params=[p.double()]), dict(exp_avgs=[m[:5]]), dict(exp_avgs=[m.half()]),
        dict(exp_avg_sqs=[v8]), dict(exp_avgs=[m8]), dict(exp_avgs=[m8], exp_avg_sqs=[v8]),
        dict(exp_avgs=[m8], exp_avg_sqs=[v8], scales=[s8[:, :2]]), dict(exp_avgs=[m8], exp_avg_sqs=[v8], scales=[s8.half()]),
        dict(exp_avgs=[m8], exp_avg_sqs=[v8], scales=[s8[0]]), dict(copies=[p[:9]]), dict(copies=[p.double()]),
        dict(copies=[p, p]), dict(counter=c.float()), dict(counter=c.cpu()), dict(counter=c[:3]), dict(max_norm=0.0),
        dict(max_norm=-1.0), dict(params=[None]),
    ]
    for kw in bad:
        with pytest.raises(AssertionError):
            step(**kw)
    for kw in (dict(lr=-1.0), dict(lr=float("nan")), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1e-8),
               dict(weight_decay=float("inf")), dict(grad_scale=float("nan"))):
        with pytest.raises(capi.Cp4Error) as e:
            step(**kw)
        assert e.value.status == capi.ERR_SHAPE
    assert c.cpu().tolist() == [0, 1, 1, 0]
    with pytest.raises(ValueError):
        optim.AdamW([torch.nn.Parameter(p)], state_bits=4)
    with pytest.raises(ValueError):
        optim.AdamW([torch.nn.Parameter(p)], betas=(0.9, 1.0))
    with pytest.raises(ValueError):
        optim.AdamW([torch.nn.Parameter(p)], max_norm=0)


def test_more_than_2_to_the_32_values(optim):
    """The last values of a tensor beyond 32-bit offsets step like those of a small one."""
    n, tail = (1 << 32) + 1027, 2048 + 3          # (the tail starts with a block of the scales: n - tail is a multiple of 256)
    assert (n - tail) % 256 == 0
    gen = torch.Generator().manual_seed(13)
    p, g = torch.randn(tail, generator=gen), gradients(gen, tail).bfloat16()
    P = torch.zeros(n, device="cuda")
    G = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    P[n - tail:], G[n - tail:] = p.cuda(), g.cuda()
    m, v, s = optim.empty_moments(P, 8)
    optim.adamw_step([P], [G], [m], [v], optim.counter(), scales=[s], **HYPER)
    want = numpy_step(p.numpy(), g.float().numpy(), np.zeros(tail, F), np.zeros(tail, F), 1, **HYPER)
    q = codes(*want[1:])
    assert np.array_equal(P[n - tail:].cpu().numpy(), want[0])
    assert np.array_equal(m[n - tail:].cpu().numpy(), q[0]) and np.array_equal(v[n - tail:].cpu().numpy(), q[1])
    assert np.array_equal(s[:, -q[2].shape[1]:].cpu().numpy(), q[2])
    assert not P[:4096].any() and not m[(1 << 32) - 5000:(1 << 32) - 3000].any()
