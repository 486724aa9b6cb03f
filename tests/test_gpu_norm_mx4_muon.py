"""Layer norm, a projection held in 4 bits with adapters beside it, and the Muon step of the adapters, one after the other."""
import pytest
import torch

pytestmark = pytest.mark.gpu
D, N, R, G, T = 200, 168, 6, 3, 75


@pytest.fixture(scope="module")
def cp4():
    import paralleltnnlayers_amd as cp4
    cp4.lib()
    return cp4


class Net(torch.nn.Module):
    def __init__(self, dtype):
        super().__init__()
        from paralleltnnlayers_amd import torch_ops
        torch.manual_seed(0)
        self.norm = torch_ops.LayerNorm(D)
        self.head = torch_ops.AdapterLinear(D, N, R, adapters=G, weight_bits=4, bias=torch.randn(N))
        with torch.no_grad():
            self.norm.weight.add_(torch.randn(D, device="cuda") / 4)
            self.norm.bias.add_(torch.randn(D, device="cuda") / 4)
            self.head.B.copy_(torch.randn(G, N, R) / 8)
        self.to(dtype)

    def forward(self, x, ids):
        return self.head(self.norm(x), ids)


def batch(dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x, dy = torch.randn(T, D, generator=g) + 0.5, torch.randn(T, N, generator=g) / 16
    return x.to("cuda", dtype), dy.to("cuda", dtype), torch.randint(-1, G, (T,), generator=g, dtype=torch.int32).cuda()


def formula(cp4, net, x, dy, ids, magnitudes):
    """(y, dx, dweight, dbias, dA, dB) in 64 bits; with ``magnitudes`` of the sums' terms instead of the terms."""
    of = (lambda t: t.double().cpu().abs()) if magnitudes else (lambda t: t.double().cpu())
    W = of(cp4.mx4_dequantize(net.head.projection()))
    A, B, w, b, bias, s = (of(t) for t in (net.head.A, net.head.B, net.norm.weight, net.norm.bias, net.head.bias, net.head.scale))
    exact = x.double().cpu()
    r = 1 / (exact.var(-1, unbiased=False, keepdim=True) + net.norm.eps).sqrt()
    h = (exact - exact.mean(-1, keepdim=True)) * r
    h = h.abs() if magnitudes else h
    z, dy, ids = h * w + b, of(dy), ids.cpu()
    y, dz, dA, dB = z @ W.T + bias, dy @ W, torch.zeros_like(A), torch.zeros_like(B)
    for a in range(G):
        m = (ids == a)[:, None]
        za, dya = z * m, dy * m
        y += s[a] * za @ A[a].T @ B[a].T
        dz += s[a] * dya @ B[a] @ A[a]
        dA[a] = s[a] * (dya @ B[a]).T @ za
        dB[a] = s[a] * dya.T @ (za @ A[a].T)
    g = dz * w
    mean, along = g.mean(-1, keepdim=True), h * (g * h).mean(-1, keepdim=True)
    dx = r * (g + mean + along if magnitudes else g - mean - along)
    return y, dx, (dz * h).sum(0), dz.sum(0), dA, dB


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_gradients_through_all_of_them(cp4, dtype):
    net = Net(dtype)
    x, dy, ids = batch(dtype)
    x.requires_grad_()
    y = net(x, ids)
    y.backward(dy)
    got = (y, x.grad, net.norm.weight.grad, net.norm.bias.grad, net.head.A.grad, net.head.B.grad)
    want, size = formula(cp4, net, x.detach(), dy, ids, False), formula(cp4, net, x.detach(), dy, ids, True)
    # relative to the sums of magnitudes: half a step of the type for each tensor that lies between the two ends - z and y, dz and
    # dx, A's output, which the matrix cores take in two roundings at most - and the result, 6 together; fp32 sums of up to
    # D + N + T terms one after the other, and a dozen steps of the norm
    off = 6 * torch.finfo(dtype).eps / 2 + (D + N + T + 12) * 2.0 ** -24
    for g, v, s, what in zip(got, want, size, ("y", "dx", "dweight", "dbias", "dA", "dB")):
        assert ((g.detach().double().cpu() - v).abs() / s).max() <= off, what


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_training_in_a_graph(cp4, dtype):
    """Steps of Muon (adapters) and AdamW (norm), eager through autograd and replayed from a graph of the plain calls."""
    from paralleltnnlayers_amd import optim

    def optimizers(net):
        return (optim.Muon([net.head.A, net.head.B], lr=0.01, weight_decay=0.1),
                optim.AdamW([net.norm.weight, net.norm.bias], lr=0.01))
    eager, graphed = Net(dtype), Net(dtype)
    graphed.load_state_dict(eager.state_dict())
    of_eager, of_graphed = optimizers(eager), optimizers(graphed)
    x, dy, ids = batch(dtype)

    def one_eager():
        for o in of_eager:
            o.zero_grad()
        eager(x, ids).backward(dy)
        for o in of_eager:
            o.step()

    def one_plain():
        h, n = graphed.head, graphed.norm
        with torch.no_grad():
            z, stats = cp4.layer_norm_forward(x, n.weight, n.bias, n.eps, keep=True)
            y, kept = cp4.adapter_forward(z, h.projection(), h.A, h.B, ids, h.scale, h.bias, keep=True)
            dz, h.A.grad, h.B.grad = cp4.adapter_backward(dy, z, h.projection(), h.A, h.B, ids, h.scale, kept)
            dx, n.weight.grad, n.bias.grad = cp4.layer_norm_backward(dz, x, n.weight, stats)
        for o in of_graphed:
            o.step()
        return y, dx
    one_eager()
    one_plain()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dx = one_plain()
    for seed in range(1, 5):
        for t, new in zip((x, dy, ids), batch(dtype, seed)):
            t.copy_(new)
        graph.replay()
        leaf = x.clone().requires_grad_()
        z = eager(leaf, ids)
        (want_dx,) = torch.autograd.grad(z, [leaf], dy)
        one_eager()
        torch.cuda.synchronize()
        assert torch.equal(y, z) and torch.equal(dx, want_dx)
        for a, b in zip(graphed.parameters(), eager.parameters()):
            assert torch.equal(a, b)


def test_backward_pass_in_a_graph(cp4):
    """Captured while an eager graph of the same leaves lives: refused.  Without one: replayed."""
    from paralleltnnlayers_amd import torch_ops
    net, linear = Net(torch.bfloat16), torch_ops.Mx4Linear(torch.randn(64, D))
    x, dy, ids = batch(torch.bfloat16)
    leaf = x.clone().requires_grad_()
    for run, most in ((lambda: net.norm(leaf), dy[:, :1]), (lambda: net.head(leaf, ids), dy[:, :1]), (lambda: linear(leaf), dy[:, :1])):
        eager = run()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="eager graph"):
            with torch.cuda.graph(graph):
                torch.autograd.grad(run(), [leaf], most.expand(-1, eager.shape[-1]).contiguous())
        del eager, graph
    torch.cuda.synchronize()
    (want,) = torch.autograd.grad(net(leaf, ids), [leaf], dy)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (got,) = torch.autograd.grad(net(leaf, ids), [leaf], dy)
    for scale in (1.0, 0.5, 2.0):
        dy.mul_(scale)
        graph.replay()
        (want,) = torch.autograd.grad(net(leaf, ids), [leaf], dy)
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_example_runs_with_all_of_them(cp4):
    import importlib.util
    import math
    import os
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "adapters.py")
    spec = importlib.util.spec_from_file_location("adapters_example", at)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    before, after, agree = example.run(users=3, steps=4, images=40, size=10, four=True)
    assert math.isfinite(before) and math.isfinite(after) and 0 <= agree <= 1
    net = example.Network(3, four=True)
    net(torch.randn(5, 3, 10, 10, device="cuda"), torch.arange(5, dtype=torch.int32, device="cuda") % 3).sum().backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in net.parameters())
