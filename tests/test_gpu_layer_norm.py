"""Layer norm: forward and backward against the formulas in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def cp4():
    import paralleltnnlayers_amd as cp4
    cp4.lib()
    return cp4


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def case(T, D, dtype, seed=0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, D, generator=g) * torch.randn(D, generator=g).exp() + shift).to(dtype).cuda()
    dy = torch.randn(T, D, generator=g).to(dtype).cuda()
    return x, dy, (1 + 0.2 * torch.randn(D, generator=g)).cuda(), (0.1 * torch.randn(D, generator=g)).cuda()


def formula(x, dy, w, b, eps):
    """y, dx, dw, db in 64 bits, and for each the sum of the magnitudes that an error is relative to."""
    x, dy = x.double().cpu(), dy.double().cpu()
    D = x.shape[1]
    w = torch.ones(D, dtype=torch.float64) if w is None else w.double().cpu()
    b = torch.zeros(D, dtype=torch.float64) if b is None else b.double().cpu()
    m = x.mean(1, keepdim=True)
    r = 1 / ((x - m).square().mean(1, keepdim=True) + eps).sqrt()
    h = (x - m) * r
    g = dy * w
    y = h * w + b
    dx = r * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    # h is off by its own rounding and by the mean's, which is one of x's size
    off_h = (h.abs() + (x.abs() + m.abs()) * r) + 1
    size = (off_h * w.abs() + b.abs(),
            r * (g.abs() + g.abs().mean(1, keepdim=True) + off_h * (g * h).abs().mean(1, keepdim=True) +
                 h.abs() * (g.abs() * off_h).mean(1, keepdim=True)),
            (dy.abs() * off_h).sum(0), dy.abs().sum(0))
    return (y, dx, (dy * h).sum(0), dy.sum(0)), size


def check(got, want, size, dtype, what, terms):
    """Each value: half a step of its type, and a few fp32 roundings of what it is a sum of.  Sums of n terms are taken in
    trees of some depth log2(n) behind runs of up to 64 in a lane, so that n roundings never add up: 64 + log2(n) of half
    a step each bound them."""
    got = got.double().cpu()
    bound = want.abs() * half_step(dtype) + size * half_step(torch.float32) * (80 + math.log2(terms + 1))
    if dtype == torch.float16:
        bound = bound + 2.0 ** -25                                   # (half a step of its smallest values)
    worst = ((got - want).abs() / bound).max()
    assert worst <= 1, (what, float(worst))


SHAPES = [(1, 1), (1, 64), (3, 7), (5, 512), (4, 513), (9, 1000), (6, 1024), (33, 1025), (2, 2048), (17, 2049),
          (13, 4096), (5, 4097), (3, 8192), (2, 8193), (3, 16384), (2, 16385), (2, 25088), (1, 32768), (3000, 96), (2500, 1001)]


@pytest.mark.parametrize("dtype", list(DTYPES), ids=str)
@pytest.mark.parametrize("T,D", SHAPES)
def test_forward_and_backward(cp4, T, D, dtype):
    x, dy, w, b = case(T, D, DTYPES[dtype])
    eps = 1e-5
    want, size = formula(x, dy, w, b, eps)
    y, stats = cp4.layer_norm_forward(x, w, b, eps, keep=True)
    got = (y,) + cp4.layer_norm_backward(dy, x, w, stats)
    for g, v, s, what, t in zip(got, want, size, ("y", "dx", "dw", "db"), (x.dtype, x.dtype, torch.float32, torch.float32)):
        check(g, v, s, t, what, max(T, D))


def test_statistics_of_rows_far_from_zero(cp4):
    x, dy, w, b = case(7, 4096, torch.float32, shift=3000.0)
    want, size = formula(x, dy, w, b, 1e-5)
    y, stats = cp4.layer_norm_forward(x, w, b, 1e-5, keep=True)
    # the mean is corrected by what it leaves: y has the error of one rounding of x, not of a sum of them
    assert ((y.double().cpu() - want[0]).abs() / size[0]).max() <= 4 * half_step(torch.float32)
    got = cp4.layer_norm_backward(dy, x, w, stats)
    for g, v, s, what in zip(got, want[1:], size[1:], ("dx", "dw", "db")):
        check(g, v, s, torch.float32, what, 4096)


def test_without_weight_or_bias_and_with_what_is_wanted(cp4):
    x, dy, w, b = case(37, 300, torch.float32)
    for weight in (None, w):
        for bias in (None, b):
            want, size = formula(x, dy, weight, bias, 1e-3)
            y, stats = cp4.layer_norm_forward(x, weight, bias, 1e-3, keep=True)
            check(y, want[0], size[0], torch.float32, "y", 300)
            for wanted in ((True, False, False), (False, True, False), (False, False, True), (True, False, True)):
                got = cp4.layer_norm_backward(dy, x, weight, stats, *wanted)
                for g, v, s, wants, what in zip(got, want[1:], size[1:], wanted, ("dx", "dw", "db")):
                    assert (g is None) == (not wants)
                    if wants:
                        check(g, v, s, torch.float32, what, 300)


@pytest.mark.parametrize("dtype", list(DTYPES), ids=str)
def test_strides_alignment_and_more_dimensions(cp4, dtype):
    x, dy, w, b = case(24, 333, DTYPES[dtype])
    y, stats = cp4.layer_norm_forward(x, w, b, keep=True)
    want = (y,) + cp4.layer_norm_backward(dy, x, w, stats)
    wide = torch.zeros(24, 777, dtype=x.dtype, device="cuda")
    wx, wdy = wide[:, 5:338], wide[:, 401:734]
    wx.copy_(x)
    wdy.copy_(dy)
    w1 = torch.cat([w[:1], w])[1:]                                   # (4 bytes off a 16-byte boundary)
    y, stats = cp4.layer_norm_forward(wx, w1, b, keep=True)
    got = (y,) + cp4.layer_norm_backward(wdy, wx, w1, stats)
    assert all(torch.equal(g, v) for g, v in zip(got, want))
    for view in (lambda t: t.view(2, 3, 4, 333), lambda t: t.t().contiguous().t(), lambda t: t.view(4, 6, 333).transpose(0, 1).contiguous().transpose(0, 1)):
        y, stats = cp4.layer_norm_forward(view(x), w, b, keep=True)
        got = (y,) + cp4.layer_norm_backward(view(dy), view(x), w, stats)
        assert y.shape == view(x).shape and got[1].shape == y.shape
        assert all(torch.equal(g.reshape(v.shape), v) for g, v in zip(got, want))


def test_no_rows(cp4):
    x = torch.zeros(0, 40, device="cuda")
    y, stats = cp4.layer_norm_forward(x, keep=True)
    dx, dw, db = cp4.layer_norm_backward(x, x, None, stats)
    assert y.shape == dx.shape == (0, 40) and not dw.any() and not db.any() and dw.shape == (40,)


@pytest.mark.parametrize("dtype", list(DTYPES), ids=str)
def test_what_is_not_finite_stays_in_its_row(cp4, dtype):
    x, dy, w, b = case(9, 700, DTYPES[dtype])
    clean, stats = cp4.layer_norm_forward(x, w, b, keep=True)
    clean_dx = cp4.layer_norm_backward(dy, x, w, stats)[0]
    x[2, 5], x[4, 699], x[6, 0] = math.inf, math.nan, -math.inf
    y, stats = cp4.layer_norm_forward(x, w, b, keep=True)
    dx, dw, db = cp4.layer_norm_backward(dy, x, w, stats)
    for t in range(9):
        if t in (2, 4, 6):
            assert y[t].isnan().all() and dx[t].isnan().all()
        else:
            assert torch.equal(y[t], clean[t]) and torch.equal(dx[t], clean_dx[t])
    assert dw.isnan().all() and db.isfinite().all()
    flat = torch.full((2, 64), 3.0, device="cuda")
    assert torch.equal(cp4.layer_norm_forward(flat), torch.zeros_like(flat))


def test_gradients_against_differences(cp4):
    from paralleltnnlayers_amd import torch_ops
    torch.manual_seed(1)
    x, w, b = (torch.randn(*s, device="cuda") for s in ((4, 48), (48,), (48,)))
    dy = torch.randn(4, 48, device="cuda")
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(torch_ops.layer_norm(*leaves), leaves, dy)
    h = 1e-2
    for k, g in enumerate(grads):
        d = torch.randn_like(leaves[k])
        step = lambda s: [t.detach() + s * h * d if i == k else t.detach() for i, t in enumerate(leaves)]  # noqa: E731
        dot = lambda y: float((y.double() * dy.double()).sum())  # noqa: E731
        diff = (dot(torch_ops.layer_norm(*step(1))) - dot(torch_ops.layer_norm(*step(-1)))) / (2 * h)
        want = float((g.double() * d.double()).sum())
        # third derivatives of h^2 / 6 and fp32 outputs (192 of some 1e-7 each) over 2 h
        assert abs(diff - want) <= 2e-2 * max(1.0, float(g.norm() * d.norm())), (k, diff, want)


@pytest.mark.parametrize("wanted", [("x",), ("w",), ("b",), ("x", "w", "b")], ids="".join)
def test_python_autograd_function_matches_the_native_one(cp4, wanted):
    from paralleltnnlayers_amd import torch_ops
    x, dy, w, b = case(10, 96, torch.bfloat16)
    results = []
    for run in (torch_ops.LayerNormFunction.apply, torch_ops.layer_norm):
        d = dict(x=x.clone(), w=w.clone(), b=b.clone())
        for k in wanted:
            d[k].requires_grad_()
        y = run(d["x"], d["w"], d["b"], 1e-5)
        results.append([y.detach(), *torch.autograd.grad(y, [d[k] for k in wanted], dy.float() if "w" in wanted else dy)])
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("there", ["", "w", "b", "wb"])
def test_gradients_of_what_is_there(cp4, there):
    """The functional form without weight or bias, natively and as a Python function, each input frozen in turn."""
    from paralleltnnlayers_amd import torch_ops
    x, dy, w, b = case(11, 70, torch.float32)
    y, stats = cp4.layer_norm_forward(x, w if "w" in there else None, b if "b" in there else None, keep=True)
    want = dict(zip("xwb", cp4.layer_norm_backward(dy, x, w if "w" in there else None, stats)))
    for run in (torch_ops.layer_norm, torch_ops.LayerNormFunction.apply):
        for frozen in ("", "x", "w", "b"):
            leaves = {k: t.clone().requires_grad_(k != frozen) for k, t in (("x", x), ("w", w), ("b", b)) if k == "x" or k in there}
            z = run(leaves["x"], leaves.get("w"), leaves.get("b"), 1e-5)
            assert torch.equal(z, y)
            if not z.requires_grad:
                continue
            z.backward(dy)
            for k, t in leaves.items():
                assert (t.grad is None) == (k == frozen)
                assert k == frozen or torch.equal(t.grad, want[k])


@pytest.mark.parametrize("T, D, ld", [(5, 333, 1 << 29), (40, 5000, 1 << 27), (300, 20000, 1 << 24)])
def test_rows_beyond_32_bit_offsets(cp4, T, D, ld):
    x, dy, w, b = case(T, D, torch.bfloat16)
    y, stats = cp4.layer_norm_forward(x, w, b, keep=True)
    want = (y,) + cp4.layer_norm_backward(dy, x, w, stats)
    room = torch.empty((T - 1) * ld + 2 * D, dtype=torch.bfloat16, device="cuda")
    assert room.numel() * 2 > 1 << 32
    wx, wdy = room.as_strided((T, D), (ld, 1)), room.as_strided((T, D), (ld, 1), D)
    wx.copy_(x)
    wdy.copy_(dy)
    y, stats = cp4.layer_norm_forward(wx, w, b, keep=True)
    got = (y,) + cp4.layer_norm_backward(wdy, wx, w, stats)
    assert all(torch.equal(g, v) for g, v in zip(got, want))


@pytest.mark.parametrize("D", [100, 3000, 9000, 20000])
def test_in_its_own_place(cp4, D):
    x, dy, w, b = case(40, D, torch.bfloat16)
    want = cp4.layer_norm_forward(x, w, b)
    assert cp4.layer_norm_forward(x, w, b, out=x) is x and torch.equal(x, want)


def test_module(cp4):
    from paralleltnnlayers_amd import torch_ops
    m = torch_ops.LayerNorm(64).bfloat16()
    assert m.weight.dtype == m.bias.dtype == torch.float32
    x = torch.randn(5, 64, device="cuda").bfloat16()
    y = m(x)
    y.backward(torch.ones_like(y))
    assert y.dtype == torch.bfloat16 and m.weight.grad.dtype == torch.float32
    assert torch.equal(torch_ops.LayerNorm(64, bias=False)(x), y)
    traced = torch.jit.trace(m, (x,), check_trace=False)
    z = torch.randn(5, 64, device="cuda").bfloat16()
    assert torch.equal(traced(z), m(z))
    leaf = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(m(leaf).float().sum(), [leaf], create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated again"):
        (g.float().square().sum() + leaf.float().sum()).backward()


def test_streams_and_graph(cp4):
    x, dy, w, b = case(300, 1001, torch.bfloat16)
    y, stats = cp4.layer_norm_forward(x, w, b, keep=True)
    want = (y,) + cp4.layer_norm_backward(dy, x, w, stats)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    y, stats = cp4.layer_norm_forward(x, w, b, keep=True, stream=side)
    got = (y,) + cp4.layer_norm_backward(dy, x, w, stats, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(g, v) for g, v in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, stats = cp4.layer_norm_forward(x, w, b, keep=True)
        got = (y,) + cp4.layer_norm_backward(dy, x, w, stats)
    for seed in range(3):
        nx, ndy, _, _ = case(300, 1001, torch.bfloat16, seed)
        x.copy_(nx)
        dy.copy_(ndy)
        graph.replay()
        z, stats = cp4.layer_norm_forward(x, w, b, keep=True)
        want = (z,) + cp4.layer_norm_backward(dy, x, w, stats)
        torch.cuda.synchronize()
        assert all(torch.equal(g, v) for g, v in zip(got, want))


def test_refusals(cp4):
    x, dy, w, b = case(4, 64, torch.float32)
    y, stats = cp4.layer_norm_forward(x, w, b, keep=True)
    bad = [lambda: cp4.layer_norm_forward(x.cpu(), w, b), lambda: cp4.layer_norm_forward(x.double(), w, b),
           lambda: cp4.layer_norm_forward(x, w[:63], b), lambda: cp4.layer_norm_forward(x, w, b.half()),
           lambda: cp4.layer_norm_forward(torch.zeros(2, 32769, device="cuda")),
           lambda: cp4.layer_norm_forward(torch.zeros(2, 0, device="cuda")),
           lambda: cp4.layer_norm_forward(x, w, b, out=torch.empty(4, 63, device="cuda")),
           lambda: cp4.layer_norm_backward(dy[:3], x, w, stats), lambda: cp4.layer_norm_backward(dy.half(), x, w, stats),
           lambda: cp4.layer_norm_backward(dy, x, w, stats[:3])]
    for call in bad:
        with pytest.raises(AssertionError):
            call()
    with pytest.raises(cp4.Cp4Error, match="eps"):
        cp4.layer_norm_forward(x, w, b, -1.0)
    with pytest.raises(cp4.Cp4Error, match="eps"):
        cp4.layer_norm_forward(x, w, b, math.nan)
