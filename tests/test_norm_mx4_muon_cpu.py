"""The C ABI of the layer norm, of 4-bit projections and of Muon without a device: symbols, and arguments that are refused
before any is touched.  And what the Python layers refuse by themselves."""
import ctypes
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ONE, ODD = 256, 257                                                  # never dereferenced: checks fail first
size_t, unsigned, pointer, integer, double = ctypes.c_size_t, ctypes.c_uint, ctypes.c_void_p, ctypes.c_int, ctypes.c_double


class Codes(ctypes.Structure):
    _fields_ = [("codes", pointer), ("scales", pointer)]


class Matrix(ctypes.Structure):
    _fields_ = ([(k, pointer) for k in ("param", "grad", "momentum", "copy")] + [("count", size_t)] +
                [(k, unsigned) for k in ("rows", "cols")] + [(k, integer) for k in ("param_dtype", "grad_dtype", "copy_dtype")])


SIGNATURES = {
    "cp4_layer_norm_forward": [size_t, unsigned, integer, pointer, size_t, pointer, pointer, ctypes.c_float, pointer, pointer, pointer],
    "cp4_layer_norm_backward": [size_t, unsigned, integer, pointer, size_t, pointer, size_t, pointer, pointer, pointer, pointer, pointer,
                                pointer, size_t, pointer],
    "cp4_mx4_quantize": [size_t, unsigned, integer, pointer, size_t, pointer, pointer, pointer],
    "cp4_mx4_dequantize": [size_t, unsigned, integer, ctypes.POINTER(Codes), pointer, pointer],
    "cp4_mx4_forward": [size_t, unsigned, unsigned, integer, pointer, size_t, ctypes.POINTER(Codes), pointer, pointer, pointer, size_t, pointer],
    "cp4_mx4_backward": [size_t, unsigned, unsigned, integer, pointer, size_t, ctypes.POINTER(Codes), pointer, pointer, size_t, pointer],
    "cp4_mx4_product": [size_t, unsigned, unsigned, integer, ctypes.POINTER(Codes), ctypes.POINTER(Codes), pointer, pointer, pointer, size_t, pointer],
    "cp4_muon_step": [ctypes.POINTER(Matrix), size_t, double, double, integer, double, double, unsigned, pointer, size_t, pointer],
    "cp4_layer_norm_backward_workspace_bytes": [size_t, unsigned],
    "cp4_mx4_forward_workspace_bytes": [size_t, unsigned, unsigned, integer],
    "cp4_mx4_backward_workspace_bytes": [size_t, unsigned, unsigned, integer],
    "cp4_mx4_product_workspace_bytes": [size_t, unsigned, unsigned],
    "cp4_muon_workspace_bytes": [ctypes.POINTER(Matrix), size_t],
}


@pytest.fixture(scope="module")
def capi():
    from paralleltnnlayers_amd import capi
    capi.lib()
    return capi


@pytest.fixture(scope="module")
def call(capi):
    """A function of the library by its name, with its signature."""
    def of(name):
        f = ctypes.CDLL(capi.lib()._name)[name]
        f.argtypes, f.restype = SIGNATURES[name], size_t if name.endswith("bytes") else integer
        return f
    return of


def declared(header):
    text = open(os.path.join(ROOT, "include", "cp4", header)).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return sorted(set(re.findall(r"\b(cp4_[a-z0-9_]+)\s*\(", text)))


@pytest.mark.parametrize("name", declared("layer_norm.h") + declared("mx4.h") + declared("muon.h"))
def test_symbol_exported(capi, name):
    assert getattr(capi.lib(), name) is not None


def test_layer_norm_arguments(capi, call):
    forward, backward = call("cp4_layer_norm_forward"), call("cp4_layer_norm_backward")

    def fwd(T=4, D=64, dtype=0, x=ONE, ldx=0, weight=ONE, bias=ONE, eps=1e-5, y=ONE, stats=ONE):
        return forward(T, D, dtype, x, ldx, weight, bias, eps, y, stats, None)

    def bwd(T=4, D=64, dtype=0, dy=ONE, lddy=0, x=ONE, ldx=0, stats=ONE, dx=ONE, dw=ONE, db=ONE, ws=ONE, room=1 << 40):
        return backward(T, D, dtype, dy, lddy, x, ldx, ONE, stats, dx, dw, db, ws, room, None)
    for bad in (dict(D=0), dict(D=32769), dict(T=(1 << 40) + 1), dict(dtype=3), dict(dtype=-1), dict(ldx=63), dict(ldx=(1 << 30) + 1), dict(x=ODD)):
        assert fwd(**bad) == bwd(**bad) == capi.ERR_SHAPE, bad
    for bad in (dict(eps=-1.0), dict(eps=float("nan")), dict(y=ODD), dict(weight=ODD + 1), dict(stats=ODD)):
        assert fwd(**bad) == capi.ERR_SHAPE, bad
    assert bwd(lddy=63) == bwd(dw=ODD) == bwd(dx=ODD) == capi.ERR_SHAPE
    assert fwd(x=None) == fwd(y=None) == bwd(dy=None) == bwd(x=None) == bwd(stats=None) == capi.ERR_NULL_POINTER
    assert bwd(T=4096, ws=None) == bwd(T=4096, ws=ODD) == bwd(T=4096, room=64) == capi.ERR_WORKSPACE
    assert fwd(T=0, x=None, y=None) == bwd(dx=None, dw=None, db=None) == 0
    need = call("cp4_layer_norm_backward_workspace_bytes")
    assert need(0, 64) == need(1, 64) == need(5, 0) == need(5, 40000) == 0 and need(5000, 64) > need(50, 64) > 0 and need(1, 20000) > 0


def test_mx4_arguments(capi, call):
    q, odd, none = Codes(ONE, ONE), Codes(ONE + 8, ONE), Codes(None, ONE)
    quantize, dequantize = call("cp4_mx4_quantize"), call("cp4_mx4_dequantize")
    for T, K, dtype, x, ld, codes, want in ((4, 0, 0, ONE, 0, ONE, capi.ERR_SHAPE), (4, (1 << 22) + 1, 0, ONE, 0, ONE, capi.ERR_SHAPE),
                                            ((1 << 26) + 1, 32, 0, ONE, 0, ONE, capi.ERR_SHAPE), (4, 32, 3, ONE, 0, ONE, capi.ERR_SHAPE),
                                            (4, 32, 0, ONE, 31, ONE, capi.ERR_SHAPE), (4, 32, 1, ODD, 0, ONE, capi.ERR_SHAPE),
                                            (4, 32, 0, ONE, 0, ONE + 8, capi.ERR_SHAPE), (4, 32, 0, None, 0, ONE, capi.ERR_NULL_POINTER),
                                            (4, 32, 0, ONE, 0, None, capi.ERR_NULL_POINTER), (0, 32, 0, None, 0, None, 0)):
        assert quantize(T, K, dtype, x, ld, codes, ONE, None) == want
    assert dequantize(4, 32, 0, none, ONE, None) == dequantize(4, 32, 0, None, ONE, None) == dequantize(4, 32, 0, q, None, None) == capi.ERR_NULL_POINTER
    assert dequantize(4, 32, 0, odd, ONE, None) == dequantize(4, 32, 0, q, ODD, None) == dequantize(4, 0, 0, q, ONE, None) == capi.ERR_SHAPE
    for name, back in (("cp4_mx4_forward", False), ("cp4_mx4_backward", True)):
        run = call(name)

        def linear(T=4, K=64, N=32, dtype=1, x=ONE, ld=0, W=q, y=ONE, ws=ONE, room=1 << 40):
            return run(T, K, N, dtype, x, ld, W, *([] if back else [ONE]), y, ws, room, None)
        for bad in (dict(K=0), dict(N=0), dict(K=(1 << 22) + 1), dict(N=(1 << 22) + 1), dict(T=(1 << 26) + 1), dict(dtype=3), dict(ld=31),
                    dict(ld=(1 << 30) + 1), dict(W=odd), dict(x=ODD), dict(y=ODD)):
            assert linear(**bad) == capi.ERR_SHAPE, bad
        for bad in (dict(x=None), dict(y=None), dict(W=None), dict(W=none)):
            assert linear(**bad) == capi.ERR_NULL_POINTER, bad
        need = call(name + "_workspace_bytes")
        assert need(8192, 4096, 4096, 1) >= 4096 * 4096 * 2 and need(0, 64, 64, 1) == need(4, 0, 64, 1) == need(4, 64, 64, 7) == 0
        for bad in (dict(ws=None), dict(ws=ODD), dict(room=1 << 20)):
            assert linear(**{**dict(T=8192, K=4096, N=4096), **bad}) == capi.ERR_WORKSPACE, bad
        assert linear(T=0, x=None, y=None, W=None) == 0
    product, need = call("cp4_mx4_product"), call("cp4_mx4_product_workspace_bytes")
    assert product(4, 64, 32, 0, odd, q, None, ONE, ONE, 1 << 40, None) == product(4, 64, 0, 0, q, q, None, ONE, ONE, 1 << 40, None) == capi.ERR_SHAPE
    assert product(4, 64, 32, 0, q, q, ODD, ONE, ONE, 1 << 40, None) == product(4, 64, 32, 5, q, q, None, ONE, ONE, 1 << 40, None) == capi.ERR_SHAPE
    assert product(4, 64, 32, 0, q, none, None, ONE, ONE, 1 << 40, None) == product(4, 64, 32, 0, q, q, None, None, ONE, 1 << 40, None) == capi.ERR_NULL_POINTER
    assert need(16, 65536, 512) >= 2 * 16 * 512 * 4 and product(16, 65536, 512, 0, q, q, None, ONE, None, 0, None) == capi.ERR_WORKSPACE


def test_adapters_in_4_bits_arguments(capi):
    L = capi.lib()
    s = ctypes.byref(capi.AdapterShape(T=4, K=32, N=24, R=4, G=2, ldx=0, ldw=0, lddy=0))
    one, q = pointer(ONE), Codes(ONE, ONE)
    fwd = lambda W, T=s, ws=one: L.cp4_adapter_mx4_forward(T, 1, one, W, one, one, one, None, None, one, None, ws, size_t(1 << 40), None)  # noqa: E731
    bwd = lambda W, T=s, ws=one: L.cp4_adapter_mx4_backward(T, 1, one, one, W, one, one, one, None, one, one, one, one, ws, size_t(1 << 40), None)  # noqa: E731
    for run in (fwd, bwd):
        assert run(None) == run(ctypes.byref(Codes(None, ONE))) == run(ctypes.byref(Codes(ONE, None))) == capi.ERR_NULL_POINTER
        assert run(ctypes.byref(Codes(ONE + 4, ONE))) == capi.ERR_SHAPE and run(ctypes.byref(q), None) == capi.ERR_NULL_POINTER
        assert run(ctypes.byref(q), ws=None) == capi.ERR_WORKSPACE


def test_muon_arguments(capi, call):
    run, need = call("cp4_muon_step"), call("cp4_muon_workspace_bytes")
    good = dict(param=ONE, grad=ONE, momentum=ONE, copy=None, count=1, rows=8, cols=16, param_dtype=0, grad_dtype=0, copy_dtype=0)

    def step(m={}, lr=0.1, momentum=0.9, decay=0.0, eps=1e-7, steps=5, ws=ONE, room=1 << 40):
        return run(Matrix(**{**good, **m}), 1, lr, momentum, 1, decay, eps, steps, ws, room, None)
    for bad in (dict(rows=65537), dict(cols=65537), dict(count=(1 << 24) + 1), dict(param_dtype=3), dict(grad_dtype=-1), dict(copy=ONE, copy_dtype=9),
                dict(grad=ODD), dict(momentum=ODD + 1), dict(param=ODD), dict(copy=ODD)):
        assert step(bad) == capi.ERR_SHAPE and need(Matrix(**{**good, **bad}), 1) == 0, bad
    for bad in (dict(lr=-1.0), dict(lr=float("inf")), dict(momentum=1.0), dict(momentum=-0.1), dict(decay=-1.0), dict(eps=0.0), dict(eps=1e-31),
                dict(eps=float("nan")), dict(steps=0), dict(steps=17)):
        assert step(**bad) == capi.ERR_SHAPE, bad
    assert step(dict(grad=None)) == run(None, 1, 0.1, 0.9, 1, 0.0, 1e-7, 5, ONE, 1 << 40, None) == capi.ERR_NULL_POINTER
    assert step(ws=None) == step(ws=ODD) == step(room=8) == capi.ERR_WORKSPACE
    for nothing in (dict(count=0), dict(rows=0), dict(cols=0)):
        assert step({**nothing, "grad": None}, ws=None, room=0) == 0
    assert run(None, 0, 0.1, 0.9, 1, 0.0, 1e-7, 5, None, 0, None) == 0
    # scratch memory: of one group of entries, however many there are
    many = (Matrix * 200)(*[Matrix(**{**good, "rows": 1024, "cols": 1024})] * 200)
    assert 0 < need(many, 200) < 2 << 30
    stack = Matrix(**{**good, "count": 1 << 24, "rows": 2, "cols": 3})
    assert 0 < need(stack, 1) < 1 << 30


def test_python_refuses(capi):
    from paralleltnnlayers_amd import optim, torch_ops
    x = torch.zeros(4, 8)
    for call in (lambda: capi.layer_norm_forward(x), lambda: capi.mx4_quantize(x), lambda: optim.orthogonalize(x),
                 lambda: capi.mx4_linear(x, capi.Mx4(x.byte(), x.byte(), 8)), lambda: torch_ops.layer_norm(x)):
        with pytest.raises(AssertionError):
            call()
    for call in (lambda: optim.Muon([torch.nn.Parameter(torch.zeros(3))]), lambda: optim.Muon([torch.nn.Parameter(x)], lr=-1.0),
                 lambda: optim.Muon([torch.nn.Parameter(x)], eps=0.0), lambda: optim.Muon([torch.nn.Parameter(x)], momentum=1.0),
                 lambda: torch_ops.AdapterLinear(8, 8, 2, device="cpu", weight_bits=3), lambda: torch_ops.Mx4Linear(x, activations=8, device="cpu"),
                 lambda: capi.mx4_linear(x, None, activations=8)):
        with pytest.raises(ValueError):
            call()
    norm = torch_ops.LayerNorm(8, device="cpu").double()
    assert norm.weight.dtype == norm.bias.dtype == torch.float32 and torch_ops.LayerNorm(8, bias=False, device="cpu").bias is None
