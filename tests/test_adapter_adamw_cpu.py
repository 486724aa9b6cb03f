"""The adapters' and AdamW's C ABI without a device: symbols, and arguments that are refused before any is touched."""
import ctypes
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ONE = ctypes.c_void_p(256)      # never dereferenced: checks fail first


@pytest.fixture(scope="module")
def capi():
    from paralleltnnlayers_amd import capi
    capi.lib()
    return capi


def declared(header):
    text = open(os.path.join(ROOT, "include", "cp4", header)).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return sorted(set(re.findall(r"\b(cp4_[a-z0-9_]+)\s*\(", text)))


@pytest.mark.parametrize("name", declared("adapter.h") + declared("adamw.h"))
def test_symbol_exported(capi, name):
    assert getattr(capi.lib(), name) is not None


def test_adapter_shapes_are_refused(capi):
    L = capi.lib()
    good = dict(T=4, K=32, N=24, R=4, G=2, ldx=0, ldw=0, lddy=0)
    assert L.cp4_adapter_forward_workspace_bytes(ctypes.byref(capi.AdapterShape(**good)), 0) == 4 * 16 * 4
    assert L.cp4_adapter_kept_bytes(ctypes.byref(capi.AdapterShape(**good)), 0) == 4 * 16 * 4
    bad = [dict(K=0), dict(N=0), dict(R=0), dict(G=0), dict(R=257), dict(G=65536), dict(K=(1 << 22) + 1),
           dict(N=(1 << 22) + 1), dict(T=(1 << 31) + 1), dict(ldx=31), dict(ldw=31), dict(lddy=23), dict(ldx=(1 << 30) + 1)]
    fwd = lambda s, dtype=0, p=[ONE] * 8: L.cp4_adapter_forward(s, dtype, *p, None, ONE, 1 << 30, None)
    bwd = lambda s, dtype=0, p=[ONE] * 8, d=(ONE, ONE, ONE): L.cp4_adapter_backward(s, dtype, *p, *d, ONE, 1 << 40, None)
    for b in bad:
        s = ctypes.byref(capi.AdapterShape(**{**good, **b}))
        assert fwd(s) == capi.ERR_SHAPE and bwd(s) == capi.ERR_SHAPE, b
        assert L.cp4_adapter_forward_workspace_bytes(s, 0) == 0
    s = ctypes.byref(capi.AdapterShape(**good))
    assert fwd(s, 3) == capi.ERR_SHAPE and bwd(s, -1) == capi.ERR_SHAPE
    assert fwd(None) == capi.ERR_NULL_POINTER and bwd(None) == capi.ERR_NULL_POINTER
    for i in (0, 1, 2, 3, 4, 7):                 # (scale and bias may be missing)
        p = [ONE] * 8
        p[i] = None
        assert fwd(s, p=p) == capi.ERR_NULL_POINTER
    odd = ctypes.c_void_p(257)
    assert L.cp4_adapter_forward(s, 1, odd, *[ONE] * 7, None, ONE, 1 << 30, None) == capi.ERR_SHAPE
    assert L.cp4_adapter_forward(s, 1, *[ONE] * 8, None, ONE, 8, None) == capi.ERR_WORKSPACE
    assert L.cp4_adapter_forward(s, 1, *[ONE] * 8, None, None, 1 << 30, None) == capi.ERR_WORKSPACE
    assert L.cp4_adapter_forward(s, 1, *[ONE] * 8, None, odd, 1 << 30, None) == capi.ERR_WORKSPACE
    assert bwd(s, d=(ONE, ONE, None)) == capi.ERR_NULL_POINTER


def test_adapter_tokens_have_a_limit(capi):
    L = capi.lib()
    need = lambda T: L.cp4_adapter_kept_bytes(ctypes.byref(capi.AdapterShape(T=T, K=32, N=24, R=4, G=2, ldx=0, ldw=0, lddy=0)), 0)
    assert need(1 << 26) == 64 << 26 and need((1 << 26) + 1) == 0


def test_adapter_workspace_grows_with_its_parts(capi):
    L = capi.lib()
    need = lambda **kw: L.cp4_adapter_backward_workspace_bytes(
        ctypes.byref(capi.AdapterShape(**{**dict(T=4096, K=1024, N=512, R=16, G=2), **kw})), 1)
    assert need() >= 4096 * 16 * 4
    assert need(R=17) > need() and need(T=0) == 0


def test_adamw_arguments_are_refused(capi):
    L = capi.lib()
    tensor = dict(param=256, grad=256, exp_avg=256, exp_avg_sq=256, scale=256, scale_sq=256, copy=None, n=10, param_dtype=0,
                  grad_dtype=0, copy_dtype=0, bits=8, group=0)
    group = dict(lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.0, counter=256)

    def step(t={}, g={}, n_groups=1, scale=1.0, most=0.0, ws=ONE, room=1 << 20, groups=None):
        ts = (capi.AdamwTensor * 1)(capi.AdamwTensor(**{**tensor, **t}))
        gs = (capi.AdamwGroup * 2)(*([capi.AdamwGroup(**{**group, **g})] * 2))
        return L.cp4_adamw_step(ts, 1, gs if groups is None else None, n_groups, scale, most, None, ws, room, None)

    for t in (dict(bits=16), dict(param_dtype=3), dict(grad_dtype=-1), dict(copy=256, copy_dtype=9), dict(group=1),
              dict(n=(1 << 40) + 1)):
        assert step(t) == capi.ERR_SHAPE, t
    for t in (dict(param=None), dict(grad=None), dict(exp_avg=None), dict(exp_avg_sq=None), dict(scale=None), dict(scale_sq=None)):
        assert step(t) == capi.ERR_NULL_POINTER, t
    for g in (dict(lr=-1.0), dict(lr=float("inf")), dict(beta1=1.0), dict(beta2=-0.1), dict(eps=-1.0),
              dict(weight_decay=float("nan")), dict(counter=260)):
        assert step(g=g) == capi.ERR_SHAPE, g
    assert step(g=dict(counter=None)) == capi.ERR_NULL_POINTER
    assert step(n_groups=2) == capi.ERR_SHAPE                        # (two groups with one counter)
    assert step(n_groups=0) == capi.ERR_NULL_POINTER and step(groups=()) == capi.ERR_NULL_POINTER
    assert step(scale=float("inf")) == capi.ERR_SHAPE and step(most=-1.0) == capi.ERR_SHAPE
    assert step(most=1.0, ws=None) == capi.ERR_WORKSPACE and step(most=1.0, room=100) == capi.ERR_WORKSPACE
    assert step(most=1.0, ws=ctypes.c_void_p(264)) == capi.ERR_WORKSPACE
    assert b"workspace" in L.cp4_last_error_message()


def test_bindings_refuse_what_is_not_on_a_device(capi):
    import torch
    from paralleltnnlayers_amd import optim, torch_ops
    x = torch.zeros(2, 4)
    with pytest.raises(AssertionError):
        capi.adapter_forward(x, torch.zeros(3, 4), torch.zeros(1, 2, 4), torch.zeros(1, 3, 2), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(AssertionError):
        torch_ops.adapter_linear(x, torch.zeros(3, 4), torch.zeros(1, 2, 4), torch.zeros(1, 3, 2), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(AssertionError):
        optim.adamw_step([x], [x], [x], [x], optim.counter("cpu"), lr=1e-3)
    with pytest.raises(ValueError):
        optim.empty_moments(x, 4)
    m, v, s = optim.empty_moments(torch.zeros(1000), 8)
    assert m.dtype == torch.int8 and v.dtype == torch.uint8 and tuple(s.shape) == (2, 4)
