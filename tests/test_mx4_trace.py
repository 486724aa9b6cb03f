"""A layer that rounds its inputs to 4 bits computes from them in a trace too."""
import pytest
import torch

from paralleltnnlayers_amd import capi, torch_ops


def without_a_device(monkeypatch, N, K, bias):
    """Such a layer on the CPU, whose products are torch's of something that each input changes."""
    layer = torch_ops.Mx4Linear.__new__(torch_ops.Mx4Linear)
    torch.nn.Module.__init__(layer)
    layer.in_features, layer.activations = K, 4
    blocks = -(-K // 32)
    layer.register_buffer("weight_codes", torch.randint(0, 256, (N, blocks * 16), dtype=torch.uint8))
    layer.register_buffer("weight_scales", torch.full((N, blocks), 127, dtype=torch.uint8))
    layer.register_buffer("bias", bias)
    W = layer.weight_codes.float()[:, :1]

    def product(x, q, bias=None, activations=None, out=None):
        assert activations == 4
        y = x.sum(-1, keepdim=True) @ W.t() + (0 if bias is None else bias)
        with torch.no_grad():
            # (as the native call's memory: not made by an operator that a trace knows)
            y = torch.from_numpy(y.numpy().copy())
            return y if out is None else fill(out, y)

    def fill(out, y):
        out.numpy()[...] = y.numpy()
        return out
    monkeypatch.setattr(capi, "mx4_linear", product)
    return layer


@pytest.mark.parametrize("bias", [False, True])
def test_traced_without_a_device(monkeypatch, bias):
    layer = without_a_device(monkeypatch, 5, 70, torch.randn(5) if bias else None)
    x, z = torch.randn(4, 70), torch.randn(9, 70)
    traced = torch.jit.trace(layer, (x,), check_trace=False)
    assert torch.equal(traced(x), layer(x)) and torch.equal(traced(z), layer(z))
    for call in (layer, traced):
        with pytest.raises((ValueError, RuntimeError), match="no gradient"):
            call(z.clone().requires_grad_()).sum().backward()
        with torch.no_grad():
            assert torch.equal(call(z.clone().requires_grad_()), layer(z))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_traced(dtype):
    capi.lib()
    torch.manual_seed(0)
    layer = torch_ops.Mx4Linear(torch.randn(48, 70), torch.randn(48), activations=4)
    network = torch.nn.Sequential(torch_ops.LayerNorm(70), layer).requires_grad_(False)
    x, z = torch.randn(20, 70, device="cuda").to(dtype), torch.randn(300, 70, device="cuda").to(dtype)
    for net in (layer, network):
        traced = torch.jit.trace(net, (x,))
        for v in (z, x, z[:1]):
            assert torch.equal(traced(v), net(v)) and traced(v).dtype == dtype
        with pytest.raises((ValueError, RuntimeError), match="no gradient"):
            traced(z.clone().requires_grad_()).sum().backward()
