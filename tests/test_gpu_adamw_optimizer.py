"""The AdamW optimizer over a training's course: who steps when, states that are saved and taken up."""
import io

import pytest
import torch

pytestmark = pytest.mark.gpu

HYPER = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.01)
SIZES = (7, 300, 1025, 33)
# which parameters have a gradient in which step: all along, from the fourth on, every other one, all but two
WHEN = ["1111111111", "0001111111", "1010101010", "1110110111"]


@pytest.fixture(scope="module")
def optim():
    from paralleltnnlayers_amd import capi, optim
    capi.lib()
    return optim


def parameters():
    gen = torch.Generator().manual_seed(1)
    return [torch.nn.Parameter(torch.randn(n, generator=gen).cuda()) for n in SIZES]


def feed(params, t):
    gen = torch.Generator().manual_seed(100 + t)
    for p, when in zip(params, WHEN):
        g = torch.randn(p.shape, generator=gen).cuda()
        p.grad = g if when[t] == "1" else None


def steps(opt, params, first, last):
    for t in range(first, last):
        feed(params, t)
        opt.step()


def near(got, want, n, hyper=HYPER):
    """n steps of both in fp32: each side rounds a step (at most lr sqrt(n) long: a root of the sum of the moments' weights)
    some sixteen times and a parameter four times a step."""
    for a, b in zip(got, want):
        a, b = a.detach().double(), b.detach().double()
        allowed = 2 * n * 2.0 ** -24 * (16 * hyper["lr"] * n ** 0.5 + 4 * (b.abs() + n * hyper["lr"]))
        assert ((a - b).abs() <= allowed).all()


def test_steps_are_each_parameters_own(optim):
    """A parameter whose first gradient comes late, or that has none now and then, steps as torch's AdamW has it."""
    P, Q = parameters(), parameters()
    ours, theirs = optim.AdamW(P, **HYPER), torch.optim.AdamW(Q, **HYPER)
    for t in range(10):
        steps(ours, P, t, t + 1)
        steps(theirs, Q, t, t + 1)
        near(P, Q, t + 1)
    for p, when in zip(P, WHEN):
        assert float(ours.state[p]["counter"][0]) == when.count("1")


def test_a_late_parameter_moves_by_its_rate(optim):
    """Its first step is lr long, not the one of moments that are a thousand steps old."""
    p, q = (torch.nn.Parameter(torch.ones(4, device="cuda")) for _ in range(2))
    opt = optim.AdamW([p, q], lr=1e-3, weight_decay=0.0)
    for _ in range(1000):
        p.grad = torch.ones_like(p)
        opt.step()
    q.grad = torch.ones_like(q)
    opt.step()
    assert torch.allclose(q, torch.full_like(q, 1 - 1e-3), rtol=0, atol=1e-6)


def test_parameters_that_step_together_share_a_count(optim):
    P = parameters()
    opt = optim.AdamW([dict(params=P[:3]), dict(params=P[3:])], **HYPER)
    count = lambda i: opt.state[P[i]]["counter"]  # noqa: E731
    for t in range(2):
        for p in P:
            p.grad = torch.ones_like(p)
        opt.step()
    assert count(0) is count(1) is count(2) and count(0) is not count(3)
    P[1].grad = None
    opt.step()
    assert count(0) is count(2) and count(0) is not count(1)
    assert [float(count(i)[0]) for i in range(4)] == [3, 2, 3, 3]
    opt.param_groups[1]["params"].append(opt.param_groups[0]["params"].pop())    # (a parameter that changes its group)
    for p in P:
        p.grad = torch.ones_like(p)
    opt.step()
    assert [float(count(i)[0]) for i in range(4)] == [4, 3, 4, 4]
    assert len({id(count(i)) for i in (0, 2, 3)}) == 3


@pytest.mark.parametrize("bits", [32, 8])
def test_a_course_that_is_taken_up_again(optim, bits):
    """Saved in the middle, with counts that have parted, and gone on from the file: the same bits."""
    P = parameters()
    kw = dict(HYPER, state_bits=bits, min_8bit_size=256, max_norm=1.0)
    opt = optim.AdamW(P, **kw)
    steps(opt, P, 0, 5)
    room = io.BytesIO()
    torch.save([[p.detach() for p in P], opt.state_dict()], room)
    steps(opt, P, 5, 10)
    room.seek(0)
    values, state = torch.load(room, weights_only=True)
    Q = [torch.nn.Parameter(v) for v in values]
    new = optim.AdamW(Q, **kw)
    new.load_state_dict(state)
    steps(new, Q, 5, 10)
    assert all(torch.equal(a, b) for a, b in zip(P, Q))
    for p, q in zip(P, Q):
        for k, t in opt.state[p].items():
            assert torch.equal(t, new.state[q][k]), k


def test_a_course_begun_with_torchs_optimizer(optim):
    Q = parameters()
    theirs = torch.optim.AdamW(Q, **HYPER)
    steps(theirs, Q, 0, 5)
    P = [torch.nn.Parameter(q.detach().clone()) for q in Q]
    ours = optim.AdamW(P, **HYPER)
    ours.load_state_dict(theirs.state_dict())
    for t in range(5, 10):
        steps(ours, P, t, t + 1)
        steps(theirs, Q, t, t + 1)
        near(P, Q, t + 1)


def test_counts_that_part_are_not_captured(optim):
    """A replay would copy the count anew each time: refused; taken before the capture, replays count on."""
    P = parameters()[:2]
    opt = optim.AdamW(P, **HYPER)
    for p in P:
        p.grad = torch.ones_like(p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step()
        P[1].grad = None
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="part here"):
            with torch.cuda.graph(graph, stream=side):
                opt.step()
        opt.step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            opt.step()
        for _ in range(3):
            graph.replay()
            side.synchronize()
    torch.cuda.current_stream().wait_stream(side)
    assert [float(opt.state[p]["counter"][0]) for p in P] == [5, 1]


def test_a_first_step_is_not_captured(optim):
    """Its moments would be zeroed in every replay: refused, and the parameter has no state then."""
    P = parameters()[:2]
    opt = optim.AdamW(P, **HYPER)
    P[0].grad = torch.ones_like(P[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step()
        P[1].grad = torch.ones_like(P[1])
        with pytest.raises(RuntimeError, match="first step"):
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
                opt.step()
        assert not opt.state.get(P[1])
        opt.step()
    torch.cuda.current_stream().wait_stream(side)
    assert [float(opt.state[p]["counter"][0]) for p in P] == [2, 1]
    first = P[1].detach() - parameters()[1].detach() * (1 - HYPER["lr"] * HYPER["weight_decay"])
    assert torch.allclose(first, torch.full_like(first, -HYPER["lr"]), rtol=0, atol=1e-6)
