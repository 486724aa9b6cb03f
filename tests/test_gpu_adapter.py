"""Low-rank adapters beside a shared projection against their formulas in 64 bits.

Bounds are sums of what each rounding can do: a sum of K products in fp32 is off by at most
(K + 8) 2^-23 of the sum of their magnitudes (one rounding a term, and a matrix instruction may cut
instead of rounding); h enters the second product as two bfloat16 parts, 2^-16 of it, in 16-bit layers;
an output is rounded once, 2^-9 (bfloat16) or 2^-12 (float16, 2^-25 near zero) of it.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ROUND = {"f32": 0.0, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
SPLIT = {"f32": 0.0, "bf16": 2.0 ** -16, "f16": 2.0 ** -16}


@pytest.fixture(scope="module")
def cp4():
    import paralleltnnlayers_amd as p
    p.lib()
    return p


def ids_of(pattern, T, G, gen):
    if pattern == "runs":                  # requests one after the other, some without an adapter
        cuts = torch.randint(1, max(2, T // 3 + 2), (T,), generator=gen)
        which = torch.randint(-1, G, (T,), generator=gen)
        ids = torch.repeat_interleave(which, cuts)[:T]
    elif pattern == "mixed":
        ids = torch.randint(-1, G, (T,), generator=gen)
    elif pattern == "one":
        ids = torch.full((T,), G - 1)
    elif pattern == "none":
        ids = torch.full((T,), -1)
    else:                                  # "outside": ids that are no adapter's
        ids = torch.tensor([-7, G, G + 5, 2 ** 31 - 1, -2 ** 31, 0])[torch.randint(0, 6, (T,), generator=gen)]
    return ids.int()


def make(dtype, T, K, N, R, G, pattern, seed=0):
    gen = torch.Generator().manual_seed(seed)
    n = lambda *s, std=1.0: (torch.randn(*s, generator=gen) * std).to(DTYPES[dtype])
    return dict(x=n(T, K), W=n(N, K, std=K ** -0.5), A=n(G, R, K, std=K ** -0.5), B=n(G, N, R, std=R ** -0.5),
                scale=0.25 + torch.rand(G, generator=gen), bias=torch.randn(N, generator=gen), dy=n(T, N),
                ids=ids_of(pattern, T, G, gen))


def formula(d, dtype, scale=True, bias=True):
    """{name: (value, bound)} of y, dx, dA and dB in 64 bits."""
    x, W, A, B, dy = (d[k].double() for k in ("x", "W", "A", "B", "dy"))
    ids, G = d["ids"].long(), A.shape[0]
    (T, K), (N, R) = x.shape, B.shape[1:]
    s = d["scale"].double() if scale else torch.ones(G, dtype=torch.float64)
    eps = 2.0 ** -23

    def product(a, b, depth):              # a [m, k], b [k, n]: value, and the bound of an fp32 sum
        return a @ b, (depth + 8) * eps * (a.abs() @ b.abs())

    y, ey = product(x, W.t(), K)
    dx, ex = product(dy, W, N)
    if bias:
        y = y + d["bias"].double()
        ey = ey + eps * y.abs()
    dA, eA = torch.zeros_like(A), torch.zeros_like(A)
    dB, eB = torch.zeros_like(B), torch.zeros_like(B)
    for a in range(G):
        at = (ids == a).nonzero().flatten()
        if not len(at):
            continue
        n = len(at)
        h, eh = product(x[at], A[a].t(), K)
        h, eh = h * s[a], (eh + 2 * eps * h.abs()) * s[a]
        dh, edh = product(dy[at], B[a], N)
        dh, edh = dh * s[a], (edh + 2 * eps * dh.abs()) * s[a]
        eh, edh = eh + SPLIT[dtype] * h.abs(), edh + SPLIT[dtype] * dh.abs()
        for out, err, p, ep, f in ((y, ey, h, eh, B[a].t()), (dx, ex, dh, edh, A[a])):
            v, e = product(p, f, R)
            out[at] += v
            err[at] += e + ep @ f.abs()
        v, e = product(dh.t(), x[at], n)
        dA[a], eA[a] = v, e + edh.t() @ x[at].abs()
        v, e = product(dy[at].t(), h, n)
        dB[a], eB[a] = v, e + dy[at].abs().t() @ eh
    out = {}
    for k, v, e in (("y", y, ey), ("dx", dx, ex), ("dA", dA, eA), ("dB", dB, eB)):
        tiny = 2.0 ** -24 if dtype == "f16" else 0.0
        out[k] = v, e + ROUND[dtype] * (v.abs() + e) + tiny + eps * v.abs()
    return out


def check(got, want, name):
    value, bound = want
    off = (got.double().cpu() - value).abs()
    worst = float((off - bound).max()) if off.numel() else 0.0
    assert worst <= 0, f"{name}: beyond its bound by {worst:.3g} (largest error {float(off.max()):.3g})"


SIZES = [  # T, K, N, R, G
    (1, 64, 64, 8, 1), (1, 1, 1, 1, 1), (2, 8, 24, 16, 3), (5, 1000, 136, 4, 7), (16, 512, 320, 16, 16),
    (17, 264, 72, 64, 2), (31, 96, 1001, 5, 64), (48, 4096, 512, 16, 40), (64, 1024, 200, 33, 5),
    (65, 33, 65, 17, 3), (100, 2048, 96, 16, 1), (130, 1001, 129, 7, 9), (200, 128, 777, 48, 4),
    (257, 320, 520, 16, 6), (300, 72, 1024, 64, 300), (513, 640, 264, 100, 3), (600, 1024, 1024, 256, 2),
    (1031, 512, 512, 16, 8),
]


@pytest.mark.parametrize("pattern", ["runs", "mixed"])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_layer_and_gradients(cp4, dtype, size, pattern):
    T, K, N, R, G = size
    d = make(dtype, T, K, N, R, G, pattern, seed=T + K)
    want = formula(d, dtype)
    g = {k: v.cuda() for k, v in d.items()}
    y, kept = cp4.adapter_forward(g["x"], g["W"], g["A"], g["B"], g["ids"], g["scale"], g["bias"], keep=True)
    check(y, want["y"], "y")
    assert torch.equal(y, cp4.adapter_forward(g["x"], g["W"], g["A"], g["B"], g["ids"], g["scale"], g["bias"]))
    dx, dA, dB = cp4.adapter_backward(g["dy"], g["x"], g["W"], g["A"], g["B"], g["ids"], g["scale"], kept)
    for k, v in (("dx", dx), ("dA", dA), ("dB", dB)):
        check(v, want[k], k)


@pytest.mark.parametrize("size", [(96, 64, 72, 40, 96), (128, 96, 136, 16, 128), (250, 136, 264, 33, 260), (310, 72, 1040, 7, 400)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_every_token_its_own_adapter(cp4, dtype, size):
    T, K, N, R, G = size
    d = make(dtype, T, K, N, R, G, "none", seed=9)
    d["ids"] = torch.randperm(G, generator=torch.Generator().manual_seed(T))[:T].int()
    want = formula(d, dtype)
    g = {k: v.cuda() for k, v in d.items()}
    y, kept = cp4.adapter_forward(g["x"], g["W"], g["A"], g["B"], g["ids"], g["scale"], g["bias"], keep=True)
    check(y, want["y"], "y")
    grads = cp4.adapter_backward(g["dy"], g["x"], g["W"], g["A"], g["B"], g["ids"], g["scale"], kept)
    for k, v in zip(("dx", "dA", "dB"), grads):
        check(v, want[k], k)


@pytest.mark.parametrize("T,G", [(17, 2), (33, 1), (40, 40), (64, 3)])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_few_tokens_of_a_wide_layer(cp4, dtype, T, G):
    """Few tokens on tiles and on the kernel of few rows, whichever the number of adapters asks for."""
    d = make(dtype, T, 1016, 9008, 12, G, "mixed", seed=T)
    want = formula(d, dtype)
    g = {k: v.cuda() for k, v in d.items()}
    y, kept = cp4.adapter_forward(g["x"], g["W"], g["A"], g["B"], g["ids"], g["scale"], g["bias"], keep=True)
    check(y, want["y"], "y")
    grads = cp4.adapter_backward(g["dy"], g["x"], g["W"], g["A"], g["B"], g["ids"], g["scale"], kept)
    for k, v in zip(("dx", "dA", "dB"), grads):
        check(v, want[k], k)


@pytest.mark.parametrize("pattern", ["one", "none", "outside"])
@pytest.mark.parametrize("size", [(1, 256, 128, 16, 4), (40, 320, 200, 8, 3), (300, 1000, 264, 20, 5)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_who_has_which_adapter(cp4, dtype, size, pattern):
    T, K, N, R, G = size
    d = make(dtype, T, K, N, R, G, pattern, seed=3)
    want = formula(d, dtype, scale=False, bias=False)
    g = {k: v.cuda() for k, v in d.items()}
    for ids in (g["ids"], g["ids"].long() + (2 ** 32 if pattern == "none" else 0)):
        y, kept = cp4.adapter_forward(g["x"], g["W"], g["A"], g["B"], ids, keep=True)
        check(y, want["y"], "y")
        grads = cp4.adapter_backward(g["dy"], g["x"], g["W"], g["A"], g["B"], ids, None, kept)
        for k, v in zip(("dx", "dA", "dB"), grads):
            check(v, want[k], k)
            if pattern == "none" and k != "dx":
                assert not v.any()


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_strides_and_offsets(cp4, dtype):
    """Rows further apart than they are long, and operands that start off 16-byte boundaries."""
    T, K, N, R, G = 70, 264, 136, 12, 3
    d = make(dtype, T, K, N, R, G, "runs", seed=5)
    want = formula(d, dtype)
    g = {k: v.cuda() for k, v in d.items()}

    def apart(t, extra, off):              # the same values in wider rows
        wide = torch.full((t.shape[0], t.shape[1] + extra), float("nan"), dtype=t.dtype, device="cuda")
        view = wide[:, off:off + t.shape[1]]
        view.copy_(t)
        return view

    def shifted(t, off):
        flat = torch.full((t.numel() + off,), float("nan"), dtype=t.dtype, device="cuda")
        flat[off:].copy_(t.flatten())
        return flat[off:].view(t.shape)

    forms = [
        dict(x=apart(g["x"], 8, 0), W=apart(g["W"], 16, 8), dy=apart(g["dy"], 24, 8)),
        dict(x=apart(g["x"], 3, 1), dy=apart(g["dy"], 1, 0)),
        dict(W=apart(g["W"], 5, 2)),
        dict(A=shifted(g["A"], 1), B=shifted(g["B"], 3)),
        dict(x=shifted(g["x"], 1), W=shifted(g["W"], 1), dy=shifted(g["dy"], 5)),
        dict(x=g["x"].t().contiguous().t(), W=g["W"].t().contiguous().t()),
        dict(scale=shifted(g["scale"], 1), bias=shifted(g["bias"], 3), ids=torch.stack([g["ids"]] * 2, 1)[:, 0]),
    ]
    for i, f in enumerate(forms):
        f = {**g, **f}
        y, kept = cp4.adapter_forward(f["x"], f["W"], f["A"], f["B"], f["ids"], f["scale"], f["bias"], keep=True)
        check(y, want["y"], f"form {i} y")
        grads = cp4.adapter_backward(f["dy"], f["x"], f["W"], f["A"], f["B"], f["ids"], f["scale"], kept)
        for k, v in zip(("dx", "dA", "dB"), grads):
            check(v, want[k], f"form {i} {k}")


@pytest.mark.parametrize("T", [3, 40, 300])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_a_spoiled_adapter_is_nobody_elses(cp4, dtype, T):
    """NaN and infinities in one adapter, and in one token, stay with them."""
    K, N, R, G = 320, 264, 16, 3
    d = make(dtype, T, K, N, R, G, "mixed", seed=7)
    d["ids"][:3] = torch.tensor([0, 1, 2])
    want = formula(d, dtype)
    g = {k: v.cuda().clone() for k, v in d.items()}
    g["A"][1, 2, 5], g["B"][1, 7, 1] = float("nan"), float("inf")
    y, kept = cp4.adapter_forward(g["x"], g["W"], g["A"], g["B"], g["ids"], g["scale"], g["bias"], keep=True)
    dx, dA, dB = cp4.adapter_backward(g["dy"], g["x"], g["W"], g["A"], g["B"], g["ids"], g["scale"], kept)
    ours = d["ids"] != 1
    for k, v in (("y", y), ("dx", dx)):
        check(v.cpu()[ours], tuple(t[ours] for t in want[k]), k)
    for k, v in (("dA", dA), ("dB", dB)):
        check(v.cpu()[[0, 2]], tuple(t[[0, 2]] for t in want[k]), k)
    assert y.cpu()[~ours].isnan().any(dim=1).all()

    g = {k: v.cuda().clone() for k, v in d.items()}
    g["x"][0], g["dy"][0] = float("nan"), float("inf")
    y, kept = cp4.adapter_forward(g["x"], g["W"], g["A"], g["B"], g["ids"], g["scale"], g["bias"], keep=True)
    dx, dA, dB = cp4.adapter_backward(g["dy"], g["x"], g["W"], g["A"], g["B"], g["ids"], g["scale"], kept)
    for k, v in (("y", y), ("dx", dx)):
        check(v.cpu()[1:], tuple(t[1:] for t in want[k]), k)
    for k, v in (("dA", dA), ("dB", dB)):
        check(v.cpu()[1:], tuple(t[1:] for t in want[k]), k)
    assert y[0].isnan().all()


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_no_tokens(cp4, dtype):
    d = {k: v.cuda() for k, v in make(dtype, 4, 64, 48, 8, 2, "runs").items()}
    e = {k: d[k][:0] for k in ("x", "dy", "ids")}
    y, kept = cp4.adapter_forward(e["x"], d["W"], d["A"], d["B"], e["ids"], d["scale"], d["bias"], keep=True)
    assert tuple(y.shape) == (0, 48)
    dx, dA, dB = cp4.adapter_backward(e["dy"], e["x"], d["W"], d["A"], d["B"], e["ids"], d["scale"], kept)
    assert tuple(dx.shape) == (0, 64) and not dA.any() and not dB.any()


def test_gradients_against_differences(cp4):
    """The layer is linear in x, in A and in B: half the difference of two points a whole direction apart is
    the gradient along it, up to the outputs' rounding."""
    from paralleltnnlayers_amd import torch_ops
    T, K, N, R, G = 90, 200, 150, 6, 4
    d = make("f32", T, K, N, R, G, "mixed", seed=11)
    bound = formula(d, "f32")["y"][1]
    g = {k: v.cuda() for k, v in d.items()}
    gen = torch.Generator().manual_seed(12)
    leaf = {k: g[k].clone().requires_grad_(True) for k in ("x", "A", "B")}
    y = torch_ops.adapter_linear(leaf["x"], g["W"], leaf["A"], leaf["B"], g["ids"], g["scale"], g["bias"])
    y.backward(g["dy"])
    for k in leaf:
        along = (torch.randn(leaf[k].shape, generator=gen) * leaf[k].detach().cpu().std()).cuda()
        ends = []
        for sign in (1, -1):
            p = {**g, k: g[k] + sign * along}
            out = torch_ops.adapter_linear(p["x"], p["W"], p["A"], p["B"], p["ids"], p["scale"], p["bias"])
            ends.append(float((out.double() * g["dy"].double()).sum()))
        by_gradient = float((leaf[k].grad.double() * along.double()).sum())
        # each end's y is off by no more than four times the bound at the middle (operands up to twice as large)
        allowed = float((4 * bound * d["dy"].double().abs()).sum()) + 1e-5 * abs(by_gradient)
        assert abs((ends[0] - ends[1]) / 2 - by_gradient) <= allowed, k


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_differentiable_layer(cp4, dtype):
    """Autograd: batches of any shape, what is not wanted, broadcast gradients."""
    from paralleltnnlayers_amd import torch_ops
    d = make(dtype, 60, 128, 96, 8, 3, "runs", seed=13)
    want = formula(d, dtype)
    g = {k: v.cuda() for k, v in d.items()}
    x3 = g["x"].view(4, 15, 128).requires_grad_(True)
    A, B = g["A"].clone().requires_grad_(True), g["B"].clone().requires_grad_(True)
    y = torch_ops.adapter_linear(x3, g["W"], A, B, g["ids"].view(4, 15), g["scale"], g["bias"])
    assert tuple(y.shape) == (4, 15, 96)
    check(y.detach().view(60, 96), want["y"], "y")
    y.backward(g["dy"].view(4, 15, 96))
    check(x3.grad.view(60, 128), want["dx"], "dx")
    check(A.grad, want["dA"], "dA")
    check(B.grad, want["dB"], "dB")
    # factors alone, input alone
    A2 = g["A"].clone().requires_grad_(True)
    torch_ops.adapter_linear(g["x"], g["W"], A2, g["B"], g["ids"], g["scale"]).backward(g["dy"])
    assert torch.equal(A2.grad, A.grad)
    x2 = g["x"].clone().requires_grad_(True)
    torch_ops.adapter_linear(x2, g["W"], g["A"], g["B"], g["ids"], g["scale"]).backward(g["dy"])
    assert torch.equal(x2.grad, x3.grad.view(60, 128))
    # a gradient that is one value broadcast
    x2.grad = None
    torch_ops.adapter_linear(x2, g["W"], g["A"], g["B"], g["ids"], g["scale"]).sum().backward()
    check(x2.grad, formula({**d, "dy": torch.ones_like(d["dy"])}, dtype)["dx"], "dx of ones")
    with torch.no_grad():
        assert not torch_ops.adapter_linear(x2, g["W"], A, B, g["ids"]).requires_grad


def test_module_starts_as_its_projection(cp4):
    from paralleltnnlayers_amd import torch_ops
    torch.manual_seed(0)
    dense = torch.nn.Linear(80, 56).cuda()
    m = torch_ops.AdapterLinear(80, 56, rank=4, adapters=3, alpha=8, weight=dense.weight, bias=dense.bias)
    x, ids = torch.randn(9, 80, device="cuda"), torch.tensor([0, 1, 2, -1, 0, 0, 2, 1, -1], device="cuda")
    assert [n for n, _ in m.named_parameters()] == ["A", "B"]
    assert torch.allclose(m(x, ids), dense(x), rtol=1e-5, atol=1e-5)
    assert float(m.scale[0]) == 2.0
    m(x, ids).square().sum().backward()
    assert m.B.grad.abs().sum() > 0 and not m.A.grad.any()         # (B is zero: nothing reaches A yet)


def test_another_stream(cp4):
    d = make("bf16", 200, 512, 384, 16, 4, "runs", seed=17)
    g = {k: v.cuda() for k, v in d.items()}
    args = [g[k] for k in ("x", "W", "A", "B", "ids", "scale", "bias")]
    y0, kept0 = cp4.adapter_forward(*args, keep=True)
    back = lambda kept, **kw: cp4.adapter_backward(g["dy"], *args[:6], kept, **kw)
    want = back(kept0)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    for _ in range(3):
        y, kept = cp4.adapter_forward(*args, keep=True, stream=st)
        got = back(kept, stream=st)
        st.synchronize()
        assert torch.equal(y, y0) and all(torch.equal(a, b) for a, b in zip(got, want))


def test_recorded_in_a_graph(cp4):
    """Every replay reads the ids anew and equals the eager result."""
    d = make("bf16", 48, 1024, 512, 16, 8, "mixed", seed=19)
    g = {k: v.cuda() for k, v in d.items()}
    args = [g[k] for k in ("x", "W", "A", "B", "ids", "scale", "bias")]

    def both():
        y, kept = cp4.adapter_forward(*args, keep=True)
        return (y, *cp4.adapter_backward(g["dy"], *args[:6], kept))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    gen = torch.Generator().manual_seed(20)
    for pattern in ("mixed", "one", "none", "runs"):
        g["ids"].copy_(ids_of(pattern, 48, 8, gen))
        g["x"].mul_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, both()):
            assert torch.equal(a, b)


def test_refusals(cp4):
    from paralleltnnlayers_amd import torch_ops
    d = {k: v.cuda() for k, v in make("f32", 6, 32, 24, 4, 2, "runs").items()}
    x, W, A, B, ids, scale, bias, dy = (d[k] for k in ("x", "W", "A", "B", "ids", "scale", "bias", "dy"))
    bad = [
        (x[:, :31], W, A, B, ids), (x, W[:, :31], A, B, ids), (x, W, A[:, :3], B, ids), (x, W, A, B[:, :23], ids),
        (x, W, A[:1], B, ids), (x, W, A, B, ids[:5]), (x, W, A, B, ids.float()), (x, W, A, B, ids.cpu()),
        (x.cpu(), W, A, B, ids), (x.half(), W, A, B, ids), (x, W, A.bfloat16(), B, ids), (x.double(), W.double(), A.double(), B.double(), ids),
        (x, W, A, B, ids, scale[:1]), (x, W, A, B, ids, scale.half()), (x, W, A, B, ids, scale, bias[:5]),
    ]
    for args in bad:
        with pytest.raises(AssertionError):
            cp4.adapter_forward(*args)
    wide = torch.zeros(2, 257, 32, device="cuda"), torch.zeros(2, 24, 257, device="cuda")
    with pytest.raises(AssertionError):
        cp4.adapter_forward(x, W, *wide, ids)
    for out in (torch.empty(6, 23, device="cuda"), torch.empty(6, 24, device="cuda", dtype=torch.float16),
                torch.empty(24, 6, device="cuda").t()):
        with pytest.raises(AssertionError):
            cp4.adapter_forward(x, W, A, B, ids, out=out)
    _, kept = cp4.adapter_forward(x, W, A, B, ids, keep=True)
    for args in ((dy[:, :5], x, W, A, B, ids, None, kept), (dy, x[:4], W, A, B, ids, None, kept),
                 (dy, x, W, A, B, ids, None, kept[:-1]), (dy, x, W, A, B, ids, None, None)):
        with pytest.raises(AssertionError):
            cp4.adapter_backward(*args)
    for frozen in (dict(W=W.clone().requires_grad_(True)), dict(bias=bias.clone().requires_grad_(True)),
                   dict(scale=scale.clone().requires_grad_(True))):
        p = {**d, **frozen}
        with pytest.raises(ValueError, match="not trained"):
            torch_ops.adapter_linear(p["x"], p["W"], p["A"], p["B"], p["ids"], p["scale"], p["bias"])


def test_example_trains_and_serves(cp4):
    """The example: a CP convolution and adapters trained by the library's AdamW, then served together."""
    import importlib.util
    import os
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "adapters.py")
    spec = importlib.util.spec_from_file_location("adapters_example", at)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    before, after, agree = module.run(users=4, steps=10, images=64)
    assert after < before
    assert agree == 1.0


@pytest.mark.parametrize("T, ld", [(5, 1 << 29), (40, 1 << 27), (300, 1 << 24)])
def test_rows_beyond_32_bit_offsets(cp4, T, ld):
    """Rows so far apart that the last ones lie beyond 2^32 bytes."""
    K, N, R, G = 264, 200, 8, 3
    d = make("bf16", T, K, N, R, G, "mixed", seed=23)
    want = formula(d, "bf16")
    g = {k: v.cuda() for k, v in d.items()}
    room = torch.empty((T - 1) * ld + 512, dtype=torch.bfloat16, device="cuda")
    assert room.numel() * 2 > 1 << 32
    x = room.as_strided((T, K), (ld, 1))
    x.copy_(g["x"])
    y, kept = cp4.adapter_forward(x, g["W"], g["A"], g["B"], g["ids"], g["scale"], g["bias"], keep=True)
    check(y, want["y"], "y")
    dy = room.as_strided((T, N), (ld, 1), 272)
    if 272 + N > 512:
        dy = room.as_strided((T, N), (ld, 1))
        x = g["x"]
    dy.copy_(g["dy"])
    for k, v in zip(("dx", "dA", "dB"), cp4.adapter_backward(dy, x, g["W"], g["A"], g["B"], g["ids"], g["scale"], kept)):
        check(v, want[k], k)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("size", [(2077, 512, 1024, 32, 5), (700, 2048, 264, 16, 4), (1500, 192, 2112, 24, 3),
                                  (4200, 130, 257, 9, 6)], ids=lambda s: "x".join(map(str, s)))
def test_every_shape_of_tile(cp4, dtype, size):
    """Batches beyond one tile, with rows left over."""
    T, K, N, R, G = size
    d = make(dtype, T, K, N, R, G, "runs", seed=29)
    want = formula(d, dtype)
    g = {k: v.cuda() for k, v in d.items()}
    y, kept = cp4.adapter_forward(g["x"], g["W"], g["A"], g["B"], g["ids"], g["scale"], g["bias"], keep=True)
    check(y, want["y"], "y")
    for k, v in zip(("dx", "dA", "dB"), cp4.adapter_backward(g["dy"], g["x"], g["W"], g["A"], g["B"], g["ids"], g["scale"], kept)):
        check(v, want[k], k)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_large_tiles(cp4, dtype):
    """The 256 x 256 tiles of both directions, on sampled rows and columns."""
    T, K, N, R, G = 4096 + 40, 2048 + 72, 4096, 16, 8
    gen = torch.Generator(device="cuda").manual_seed(31)
    n = lambda *s, std=1.0: (torch.randn(*s, device="cuda", generator=gen) * std).to(DTYPES[dtype])
    x, W, A, B, dy = n(T, K), n(N, K, std=K ** -0.5), n(G, R, K, std=K ** -0.5), n(G, N, R, std=R ** -0.5), n(T, N)
    ids = ids_of("runs", T, G, torch.Generator().manual_seed(32))
    scale = torch.full((G,), 0.5, device="cuda")
    y, kept = cp4.adapter_forward(x, W, A, B, ids.cuda(), scale, keep=True)
    dx = cp4.adapter_backward(dy, None, W, A, B, ids.cuda(), scale, want_factors=False)[0]
    rows = torch.cat([torch.arange(0, T, 97), torch.arange(T - 45, T)])
    d = dict(x=x.cpu()[rows], W=W.cpu(), A=A.cpu(), B=B.cpu(), dy=dy.cpu()[rows], ids=ids[rows], scale=scale.cpu(),
             bias=torch.zeros(N))
    want = formula(d, dtype, bias=False)
    check(y.cpu()[rows], want["y"], "y")
    check(dx.cpu()[rows], want["dx"], "dx")
