"""Layer norm and projections in 4 bits as a program uses them: hooked, checkpointed, transformed, given outputs."""
import pytest
import torch

pytestmark = pytest.mark.gpu
T, K, N = 10, 64, 48


@pytest.fixture(scope="module")
def cp4():
    import paralleltnnlayers_amd as cp4
    cp4.lib()
    return cp4


def layers(cp4):
    """name: (a call, its leaves)."""
    from paralleltnnlayers_amd import torch_ops
    torch.manual_seed(0)
    norm = torch_ops.LayerNorm(K)
    with torch.no_grad():
        norm.weight.normal_()
        norm.bias.normal_()
    dense = torch_ops.Mx4Linear(torch.randn(N, K), torch.randn(N))
    adapter = torch_ops.AdapterLinear(K, N, 8, adapters=3, bias=torch.randn(N), weight_bits=4)
    with torch.no_grad():
        adapter.B.normal_()
    ids = torch.tensor([0, 1, 2, -1, 2, 2, 1, 0, 0, 1], device="cuda", dtype=torch.int32)
    return {"norm": (norm, list(norm.parameters())), "dense": (dense, []), "adapter": (lambda x: adapter(x, ids), [adapter.A, adapter.B])}


def batch():
    return torch.randn(T, K, generator=torch.Generator().manual_seed(1)).cuda()


def gradients(run, leaves, dy=None):
    x = batch().requires_grad_()
    y = run(x)
    return torch.autograd.grad(y, [x, *leaves], torch.ones_like(y) if dy is None else dy)


@pytest.mark.parametrize("name", ["norm", "dense", "adapter"])
def test_saved_tensor_hooks_and_checkpoints(cp4, name):
    from torch.utils.checkpoint import checkpoint
    run, leaves = layers(cp4)[name]
    want = gradients(run, leaves)

    def offloaded(x):
        with torch.autograd.graph.save_on_cpu():
            return run(x)
    for other in (offloaded, lambda x: checkpoint(run, x, use_reentrant=False)):
        assert all(torch.equal(a, b) for a, b in zip(gradients(other, leaves), want))
    y = run(batch())
    one = gradients(run, leaves, torch.ones(1, device="cuda").expand_as(y))          # (dy as a sum leaves it)
    assert all(torch.equal(a, b) for a, b in zip(one, want))


@pytest.mark.parametrize("name", ["norm", "dense", "adapter"])
def test_what_hooks_spoil_is_refused(cp4, name):
    """Each saved tensor given back in another type, shorter, or on the host: an error, never a gradient of it."""
    run, leaves = layers(cp4)[name]
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (saved.append(t), t)[1], lambda t: t):
        run(batch().requires_grad_())
    spoils = [lambda t: t.double() if t.is_floating_point() else t.float(), lambda t: t[:-1], lambda t: t.cpu()]
    for i, t in enumerate(saved):
        for spoil in spoils:
            count = iter(range(100))
            with torch.autograd.graph.saved_tensors_hooks(lambda u: spoil(u) if next(count) == i else u, lambda u: u):
                y = run(batch().requires_grad_())
            with pytest.raises(AssertionError):
                y.sum().backward()


@pytest.mark.parametrize("name", ["norm", "dense", "adapter"])
def test_transforms_are_refused(cp4, name):
    """The library sees memory, not batched or wrapped tensors: an error, never a result."""
    import torch.autograd.forward_ad as fwd
    run, leaves = layers(cp4)[name]
    x = batch()
    both = torch.stack([x, x])
    leaf = x.clone().requires_grad_()
    y = run(leaf)

    def dual():
        with torch.no_grad(), fwd.dual_level():
            run(fwd.make_dual(x, torch.ones_like(x)))
    with torch.no_grad():
        calls = [lambda: torch.vmap(run)(both)]
    calls += [dual, lambda: torch.func.grad(lambda t: run(t).sum())(x), lambda: torch.func.jvp(run, (x,), (x,)),
              lambda: torch.autograd.grad(y, leaf, torch.stack([torch.ones_like(y)] * 2), is_grads_batched=True)]
    for call in calls:
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()


def test_raw_calls_refuse_transforms(cp4):
    x, w = batch(), torch.ones(K, device="cuda")
    q = cp4.mx4_quantize(torch.randn(N, K, device="cuda"))
    from paralleltnnlayers_amd import optim
    _, stats = cp4.layer_norm_forward(x, w, keep=True)
    both = lambda t: torch.stack([t, t])  # noqa: E731
    for call in (lambda: torch.vmap(lambda t: cp4.layer_norm_forward(t, w))(both(x)), lambda: torch.vmap(lambda t: cp4.layer_norm_forward(x, t))(both(w)),
                 lambda: torch.vmap(lambda t: cp4.layer_norm_backward(t, x, w, stats)[0])(both(x)),
                 lambda: torch.vmap(lambda t: cp4.mx4_quantize(t).codes)(both(x)), lambda: torch.vmap(lambda t: cp4.mx4_linear(t, q))(both(x)),
                 lambda: torch.vmap(lambda t: cp4.mx4_linear(t, q, activations=4))(both(x)),
                 lambda: torch.vmap(lambda t: cp4.mx4_linear(x, cp4.Mx4(t, q.scales, K)))(both(q.codes)),
                 lambda: torch.vmap(lambda t: cp4.mx4_dequantize(cp4.Mx4(t, q.scales, K)))(both(q.codes)),
                 lambda: torch.vmap(lambda t: cp4.mx4_linear_backward(t, q))(both(torch.ones(T, N, device="cuda"))),
                 lambda: torch.vmap(optim.orthogonalize)(both(x))):
        with pytest.raises((RuntimeError, NotImplementedError, AssertionError)):
            call()


def test_out_is_written(cp4):
    """A result that goes into a tensor autograd has saved is noticed by its backward pass."""
    x = batch()
    q = cp4.mx4_quantize(torch.randn(N, K, device="cuda"))
    from paralleltnnlayers_amd import optim
    for shape, call in (((T, K), lambda out: cp4.layer_norm_forward(x, out=out)), ((T, N), lambda out: cp4.mx4_linear(x, q, out=out)),
                        ((T, N), lambda out: cp4.mx4_linear(x, q, activations=4, out=out)), ((N, K), lambda out: cp4.mx4_dequantize(q, out=out)),
                        ((T, K), lambda out: optim.orthogonalize(x, out=out))):
        out = torch.zeros(shape, device="cuda")
        leaf = torch.ones(shape, device="cuda", requires_grad=True)
        loss = (leaf * out).sum()
        assert call(out) is out and out.any()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
        with torch.inference_mode():
            made = torch.empty(shape, device="cuda")
            call(made)
        assert torch.equal(made, out)


def test_rows_whose_squares_are_infinite(cp4):
    """Finite rows beyond 1e19 from their mean: bias in y, 0 in dx; others are not touched by them."""
    for dtype in (torch.float32, torch.bfloat16):
        x, dy = batch().to(dtype), torch.randn(T, K, device="cuda").to(dtype)
        w, b = torch.randn(K, device="cuda"), torch.randn(K, device="cuda")
        want, stats = cp4.layer_norm_forward(x, w, b, keep=True)
        clean = cp4.layer_norm_backward(dy, x, w, stats)[0]
        x[3] = 1e25
        x[3, ::2] = -1e25
        y, stats = cp4.layer_norm_forward(x, w, b, keep=True)
        dx = cp4.layer_norm_backward(dy, x, w, stats)[0]
        assert torch.equal(y[3], b.to(dtype)) and not dx[3].any()
        rest = [t for t in range(T) if t != 3]
        assert torch.equal(y[rest], want[rest]) and torch.equal(dx[rest], clean[rest])
