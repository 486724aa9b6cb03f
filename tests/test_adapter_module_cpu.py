"""The adapters' module without a device: what conversions of a network do to it."""
import pytest
import torch

from paralleltnnlayers_amd import torch_ops


def module(**kw):
    torch.manual_seed(0)
    bias = torch.randn(6)                        # (values that 16 bits do not have)
    return torch_ops.AdapterLinear(8, 6, rank=2, adapters=3, alpha=0.7, bias=bias, device="cpu", **kw), bias


@pytest.mark.parametrize("convert", [lambda m: m.bfloat16(), lambda m: m.half(), lambda m: m.to(torch.bfloat16),
                                     lambda m: torch.nn.Sequential(m).half()[0], lambda m: m.half().float()],
                         ids=["bfloat16", "half", "to", "network", "and back"])
def test_scales_and_bias_stay_as_they_are(convert):
    m, bias = module()
    scale = m.scale.clone()
    m = convert(m)
    assert m.weight.dtype == m.A.dtype == m.B.dtype != torch.float64
    assert m.scale.dtype == m.bias.dtype == torch.float32
    assert torch.equal(m.scale, scale) and torch.equal(m.bias, bias)
    assert list(dict(m.named_buffers())) == ["weight", "bias", "scale"]


def test_other_moves_are_torchs():
    m, _ = module()
    m.to("meta")
    assert m.scale.device.type == m.bias.device.type == m.weight.device.type == "meta"
    m.to_empty(device="cpu")
    assert m.scale.dtype == torch.float32 and m.bias.device.type == "cpu"
    assert torch_ops.AdapterLinear(8, 6, rank=2, device="cpu").half().bias is None


@pytest.mark.parametrize("dtype", [torch.float16, torch.float64])
def test_another_default_type(dtype):
    torch.set_default_dtype(dtype)
    try:
        m = torch_ops.AdapterLinear(8, 6, rank=2, adapters=3, device="cpu")
    finally:
        torch.set_default_dtype(torch.float32)
    assert m.scale.dtype == m.weight.dtype == m.A.dtype == m.B.dtype == torch.float32
