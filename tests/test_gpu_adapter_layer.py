"""``adapter_linear`` and its module as a program uses them: traced, converted, hooked, differentiated."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from paralleltnnlayers_amd import capi, torch_ops
    capi.lib()
    return torch_ops


def small(ops, **kw):
    """A module whose adapters are not nothing, a batch and its ids."""
    torch.manual_seed(3)
    layer = ops.AdapterLinear(64, 48, 8, adapters=3, bias=torch.randn(48), **kw)
    with torch.no_grad():
        layer.B.copy_(torch.randn(layer.B.shape))
    x = torch.randn(10, 64, device="cuda").to(layer.A.dtype)
    return layer, x, torch.tensor([0, 1, 2, -1, 2, 2, 1, 0, 0, 1], device="cuda", dtype=torch.int32)


@pytest.mark.parametrize("grad", [True, False], ids=["training", "serving"])
def test_traced_layer_computes_from_its_inputs(ops, grad):
    """A trace holds the layer as an operator: run on another batch and other ids it gives their result."""
    layer, x, ids = small(ops)

    class Program(torch.nn.Module):
        """(with something that depends on x by itself, so that tracing would not notice a constant part)"""
        def __init__(self):
            super().__init__()
            self.layer = layer

        def forward(self, x, ids):
            return self.layer(x, ids) + x[:, :48]

    program = Program()
    with torch.set_grad_enabled(grad):
        traced = torch.jit.trace(program, (x, ids), check_trace=False)
        for other, which in ((torch.randn_like(x), ids), (x, ids.flip(0).contiguous()), (torch.randn_like(x), ids.long())):
            assert torch.equal(traced(other, which), program(other, which))


def test_traced_module_has_its_own_gradients(ops):
    layer, x, ids = small(ops)
    traced = torch.jit.trace(layer, (x, ids), check_trace=False)
    dy = torch.randn(10, 48, device="cuda")
    grads = []
    for run in (layer, traced):
        leaf = x.clone().requires_grad_()
        layer.zero_grad()
        run(leaf, ids).backward(dy)
        grads.append([leaf.grad, layer.A.grad, layer.B.grad])
    assert all(torch.equal(a, b) for a, b in zip(*grads))


@pytest.mark.parametrize("wanted", [("x",), ("A",), ("x", "B"), ("x", "A", "B")], ids="".join)
def test_python_autograd_function_matches_the_native_one(ops, wanted):
    layer, x, ids = small(ops)
    dy = torch.randn(10, 48, device="cuda")
    results = []
    for run in (ops.AdapterLinearFunction.apply, ops.adapter_linear):
        d = dict(x=x.clone(), A=layer.A.detach().clone(), B=layer.B.detach().clone())
        for k in wanted:
            d[k].requires_grad_()
        y = run(d["x"], layer.weight, d["A"], d["B"], ids, layer.scale, layer.bias)
        results.append([y.detach(), *torch.autograd.grad(y, [d[k] for k in wanted], dy)])
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_what_is_frozen_is_refused_in_a_trace(ops):
    layer, x, ids = small(ops)
    for frozen in (layer.weight, layer.scale, layer.bias):
        frozen.requires_grad_()
        with pytest.raises(ValueError, match="not trained"):
            torch.jit.trace(layer, (x, ids), check_trace=False)
        frozen.requires_grad_(False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
def test_converted_module(ops, dtype):
    """A converted network's layer runs, forward and backward: as one that was made of that type."""
    layer, x, ids = small(ops)
    made = ops.AdapterLinear(64, 48, 8, adapters=3, weight=layer.weight, bias=layer.bias, dtype=dtype)
    with torch.no_grad():
        made.A.copy_(layer.A)
        made.B.copy_(layer.B)
    layer.to(dtype)
    dy = torch.randn(10, 48, device="cuda").to(dtype)
    results = []
    for m in (layer, made):
        leaf = x.to(dtype).requires_grad_()
        y = m(leaf, ids)
        results.append([y.detach(), *torch.autograd.grad(y, [leaf, m.A, m.B], dy)])
    assert results[0][0].dtype == dtype
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("traced", [False, True], ids=["native", "python"])
def test_gradients_are_not_differentiated_again(ops, traced):
    """create_graph gives the same gradients; a derivative of one of them is refused, not taken as zero."""
    layer, x, ids = small(ops)
    apply = ops.AdapterLinearFunction.apply if traced else ops.adapter_linear

    def grads(**kw):
        leaf = x.clone().requires_grad_()
        y = apply(leaf, layer.weight, layer.A, layer.B, ids, layer.scale, layer.bias)
        return leaf, torch.autograd.grad(y.sum(), [leaf, layer.A, layer.B], **kw)

    _, want = grads()
    leaf, got = grads(create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for g in got:
        # (what else the loss consists of must not hide it)
        with pytest.raises(RuntimeError, match="differentiated again"):
            (g.square().sum() + leaf.sum() + layer.A.sum()).backward(retain_graph=True)
    assert not want[0].requires_grad


def test_out_is_written(ops):
    """A result that goes into a tensor autograd has saved is noticed by its backward pass."""
    import paralleltnnlayers_amd as cp4
    layer, x, ids = small(ops)
    args = x, layer.weight, layer.A.detach(), layer.B.detach(), ids, layer.scale, layer.bias
    out = torch.zeros(10, 48, device="cuda")
    leaf = torch.ones(10, 48, device="cuda", requires_grad=True)
    loss = (leaf * out).sum()
    y = cp4.adapter_forward(*args, out=out)
    assert y is out and torch.equal(out, cp4.adapter_forward(*args))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():                 # (a tensor without a version)
        made = torch.empty(10, 48, device="cuda")
        cp4.adapter_forward(*args, out=made)
    assert torch.equal(made, out)


@pytest.mark.parametrize("stride", [(1 << 30) + 8, 0, 63], ids=["far", "none", "short"])
def test_a_single_row_has_no_stride(ops, stride):
    """The last token of a long sequence: one row, whatever lies between it and the next that is not there."""
    import paralleltnnlayers_amd as cp4
    layer, x, ids = small(ops)
    factors = layer.A.detach(), layer.B.detach(), ids[:1], layer.scale
    dy = torch.randn(1, 48, device="cuda")
    row, drow = x[:1].as_strided((1, 64), (stride, 1)), dy.as_strided((1, 48), (stride, 1))
    one = layer.weight[:1].as_strided((1, 64), (stride, 1))
    want, kept = cp4.adapter_forward(x[:1], layer.weight, *factors, layer.bias, keep=True)
    assert torch.equal(cp4.adapter_forward(row, layer.weight, *factors, layer.bias), want)
    grads = [cp4.adapter_backward(d, r, layer.weight, *factors, kept) for d, r in ((dy, x[:1]), (drow, row))]
    assert all(torch.equal(a, b) for a, b in zip(*grads))
    narrow = factors[0], factors[1][:, :1].contiguous(), *factors[2:]
    assert torch.equal(cp4.adapter_forward(row, one, *narrow), cp4.adapter_forward(x[:1], layer.weight[:1], *narrow))


def test_saved_tensor_hooks_see_what_the_layer_saves(ops):
    """Offloading the saved tensors changes nothing; what is saved is the operands and h."""
    layer, x, ids = small(ops)
    dy = torch.randn(10, 48, device="cuda")

    def grads(run):
        leaf = x.clone().requires_grad_()
        return torch.autograd.grad(run(leaf), [leaf, layer.A, layer.B], dy)

    def offloaded(leaf):
        with torch.autograd.graph.save_on_cpu():
            return layer(leaf, ids)

    want = grads(lambda leaf: layer(leaf, ids))
    assert all(torch.equal(a, b) for a, b in zip(grads(offloaded), want))
    shapes = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (shapes.append(tuple(t.shape)), t)[1], lambda t: t):
        layer(x.clone().requires_grad_(), ids)
    h = (10 * 16,)                               # (10 tokens, rank 8 in rows of 16)
    assert sorted(shapes) == sorted([tuple(t.shape) for t in (x, layer.weight, layer.A, layer.B, ids, layer.scale)] + [h])


def test_what_hooks_spoil_is_refused(ops):
    """h given back in another type is no h: an error, never a gradient of it."""
    layer, x, ids = small(ops)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.double() if t.shape == (160,) else t, lambda t: t):
        y = layer(x, ids)
    with pytest.raises(AssertionError, match="kept"):
        y.sum().backward()


def test_forward_mode_tangents_are_refused(ops):
    import torch.autograd.forward_ad as fwd
    layer, x, ids = small(ops)
    with torch.no_grad(), fwd.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError)):
            layer(fwd.make_dual(x, torch.ones_like(x)), ids)


def test_functional_transforms_are_refused(ops):
    """The library sees memory, not batched or wrapped tensors: an error, never a result."""
    import paralleltnnlayers_amd as cp4
    layer, x, ids = small(ops)
    W, A, B, s = layer.weight, layer.A.detach(), layer.B.detach(), layer.scale
    both = lambda t: torch.stack([t, t])  # noqa: E731
    _, kept = cp4.adapter_forward(x, W, A, B, ids, keep=True)
    dy = torch.randn(10, 48, device="cuda")
    with torch.no_grad():
        calls = [lambda: torch.vmap(lambda t: layer(t, ids))(both(x)), lambda: torch.vmap(lambda t: layer(x, t))(both(ids)),
                 lambda: torch.vmap(lambda t: layer(x, t))(both(ids.long())),
                 lambda: torch.vmap(lambda t: cp4.adapter_forward(x, W, t, B, ids))(both(A)),
                 lambda: torch.vmap(lambda t: cp4.adapter_forward(x, W, A, B, ids, t))(both(s)),
                 lambda: torch.vmap(lambda t: cp4.adapter_backward(t, x, W, A, B, ids, kept=kept)[0])(both(dy))]
    leaf = x.clone().requires_grad_()
    y = layer(leaf, ids)
    calls += [lambda: torch.func.grad(lambda t: layer(t, ids).sum())(x),
              lambda: torch.func.jvp(lambda t: layer(t, ids), (x,), (x,)),
              lambda: torch.autograd.grad(y, leaf, both(dy), is_grads_batched=True)]
    for call in calls:
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()
