"""PyTorch autograd binding of the fused CP4 Conv2d C ABI.

Stands where the reference registers its TensorFlow custom op
(Kernels/cp4_conv_nchw.cc:6-108, ``Cp4Conv2dNchw``: input + four factor
tensors -> output, NCHW): a ``torch.autograd.Function`` whose forward, input
gradient and factor gradients are the three passes of ``libcp4conv.so``.
PyTorch only owns the tensors and the stream; all arithmetic is in the HIP
library, and there is no eager fallback.

Factor layout is the C ABI's: FK [T,R], FC [C,R], FH [Y,R], FW [X,R].
For "same" padding at stride 1 (2*pad = Y-1 = X-1) the reference's three passes
run as they are; that is the only case in which its backward-data formula
(flipped taps at offset +y-pad, Cuda_kernels/cp4Conv2dBackwardData.cu:79-87) is
the adjoint of its forward.  Strides and every other padding go through the
library's geometry entry points (cp4_conv2d_forward_ex and its exact gradients).

Launches are asynchronous.  A producer / consumer kernel whose wait between waves
runs out ends early and leaves its output incomplete; the library records that per
device and reports it from ``cp4_device_status``, which synchronises the stream.
``check_device()`` is that call: use it wherever the training loop synchronises
anyway (reading the loss, a checkpoint).  ``set_device_checks(True)`` - or the
environment variable ``CP4_CHECK_DEVICE=1`` - makes every backward pass of the
Functions below end with it, at the price of one synchronisation per layer and step.
"""
import os

import torch

from . import capi


def set_device_checks(on):
    """Check the device's fault record at the end of every backward pass (synchronises)."""
    global _check_every_backward
    _check_every_backward = bool(on)
    if not isinstance(capi._native, capi._Missing):
        capi._native.set_check_backward(_check_every_backward)


set_device_checks(os.environ.get("CP4_CHECK_DEVICE", "0") not in ("", "0"))


def check_device(stream=None):
    """Synchronises ``stream`` and raises ``capi.Cp4Error`` (ERR_DEVICE) if a kernel of
    the library gave up a wait since the last check: outputs computed since then are
    incomplete.  The record is cleared."""
    capi.device_status(stream)


def _after_backward():
    if _check_every_backward:
        capi.device_status()


class CP4Conv2dFunction(torch.autograd.Function):
    """y = act(cp4conv2d(x, FK, FC, FH, FW, pad) + bias) as a Python autograd function, forward
    and backward each one call of the library's layer entry points.  ``cp4_conv2d`` runs the
    native one (csrc/torch/binding.cpp); this one stands for it where a call has to be seen
    as an operator: in a trace.

    A bfloat16 or float16 ``x`` selects the library's 16-bit activations (y and the input
    gradient are of x's type then; factors, bias and their gradients stay float32); shapes
    those do not take run on widened copies.
    """

    @staticmethod
    def forward(ctx, x, FK, FC, FH, FW, pad, bias=None, activation=None):
        if 2 * pad + 1 != FH.shape[0] or 2 * pad + 1 != FW.shape[0]:
            raise ValueError("autograd binding needs 2*pad = Y-1 = X-1 (the reference's "
                             "backward-data pass is the adjoint only then)")
        x = x.contiguous()
        if x.dtype not in (torch.bfloat16, torch.float16):
            x = x.float()
        return _layer_forward(ctx, x, FK, FC, FH, FW, pad, None, bias, activation)

    @staticmethod
    def backward(ctx, dy):
        return _layer_backward(ctx, dy)


class CP4Conv2dGeometryFunction(torch.autograd.Function):
    """The same for a layer with a stride, explicit padding or an output plane of its own
    (``geom``: a ``capi.Geometry``; float32)."""

    @staticmethod
    def forward(ctx, x, FK, FC, FH, FW, geom, bias=None, activation=None):
        return _layer_forward(ctx, x.contiguous().float(), FK, FC, FH, FW, 0, geom, bias,
                              activation)

    @staticmethod
    def backward(ctx, dy):
        return _layer_backward(ctx, dy)


def _layer_forward(ctx, x, FK, FC, FH, FW, pad, geom, bias, activation):
    FK, FC, FH, FW = (t.contiguous().float() for t in (FK, FC, FH, FW))
    if bias is not None:
        bias = bias.contiguous().float()
    s = capi.shape_for(x.shape, FK, FC, FH, FW, pad)
    y = capi.layer_forward(s, geom, x, FK, FC, FH, FW, bias, activation)
    ctx.shape, ctx.geom, ctx.activation = s, geom, activation
    ctx.save_for_backward(x, FK, FC, FH, FW, y if capi.ACTIVATIONS[activation] == 1 else None)
    return y


def _layer_backward(ctx, dy):
    x, FK, FC, FH, FW, y = ctx.saved_tensors
    need = ctx.needs_input_grad
    # create_graph: the bias gradient is linear in dy and stays differentiable
    bias_graph = need[6] and torch.is_grad_enabled() and dy.requires_grad
    dx, grads, dbias = capi.layer_backward(
        ctx.shape, ctx.geom, x, y, dy.contiguous().to(x.dtype), FK, FC, FH, FW, ctx.activation,
        want_dx=need[0], want_factors=any(need[1:5]), want_bias=need[6] and not bias_graph)
    if bias_graph:
        dbias = (dy if y is None else dy * (y > 0)).float().sum(dim=(0, 2, 3))
    grads = tuple(g if n else None for g, n in zip(grads, need[1:5]))
    _after_backward()
    return (dx,) + grads + (None, dbias, None)


def _traced_layer(x, FK, FC, FH, FW, pad, bias, activation, stride, padding):
    if padding is None:
        padding = pad
    y_taps, x_taps = FH.shape[0], FW.shape[0]
    if stride == 1 and (
            (isinstance(padding, int) and 2 * padding + 1 == y_taps == x_taps) or
            (padding == "same" and y_taps == x_taps and y_taps % 2 == 1)):
        return CP4Conv2dFunction.apply(x, FK, FC, FH, FW, y_taps // 2, bias, activation)
    geom = capi.geometry(capi.shape_for(x.shape, FK, FC, FH, FW, 0), stride, padding)
    return CP4Conv2dGeometryFunction.apply(x, FK, FC, FH, FW, geom, bias, activation)


def cp4_conv2d(x, FK, FC, FH, FW, pad, bias=None, activation=None, stride=1, padding=None):
    """Functional form: differentiable fused CP4 convolution (NCHW), with the
    optional bias [T] and activation ("relu") fused into the forward stores.

    ``pad`` zeros on every side, stride 1 and 2*pad = Y - 1 is the reference's own
    layer and runs its three passes (bfloat16 activations included).  A ``stride``,
    ``padding`` = "same" (the framework's rule of the reference's Python layers,
    test/layers.py:264-279: out = ceil(in / stride), on even sizes one more zero
    after the image than before it), "valid", an int or an (h, w) pair run the
    strided kernels: only the kept outputs are computed.
    """
    # torch.jit.trace records operators: the native call would leave a constant in the graph
    run = capi._native.layer if torch._C._get_tracing_state() is None else _traced_layer
    return run(x, FK, FC, FH, FW, pad, bias, activation, stride, padding)


class CP4Conv2d(torch.nn.Module):
    """A rank-R CP4-decomposed convolution layer, "same" padding.

    Equivalent dense filter: K[t,c,y,x] = sum_r FK[t,r] FC[c,r] FH[y,r] FW[x,r]
    (Cuda_kernels/Utils.cu:55-62).  Factors start as normal(0, s) with s chosen
    so that the recomposed filter has the variance of a Kaiming-normal dense
    filter of the same shape.
    """

    def __init__(self, in_channels, out_channels, kernel_size, rank, device="cuda", bias=False,
                 activation=None, stride=1, padding=None):
        super().__init__()
        if kernel_size % 2 != 1 and padding is None:
            raise ValueError("kernel_size must be odd for the default padding")
        self.pad = kernel_size // 2
        self.padding = padding
        fan_in = in_channels * kernel_size * kernel_size
        # Var[K] = R * s^8 for four independent N(0, s^2) factors; target 2 / fan_in
        s = (2.0 / (fan_in * rank)) ** 0.125
        mk = lambda d: torch.nn.Parameter(torch.randn(d, rank, device=device) * s)
        self.FK, self.FC = mk(out_channels), mk(in_channels)
        self.FH, self.FW = mk(kernel_size), mk(kernel_size)
        self.bias = torch.nn.Parameter(torch.zeros(out_channels, device=device)) if bias else None
        self.activation = activation
        self.stride = stride

    def forward(self, x):
        return cp4_conv2d(x, self.FK, self.FC, self.FH, self.FW, self.pad, self.bias,
                          self.activation, self.stride, self.padding)

    @staticmethod
    def check_device(stream=None):
        """See ``check_device``: call where the loop synchronises anyway."""
        check_device(stream)

    def dense_filter(self):
        """The recomposed [T,C,Y,X] filter (on the device, through cp4_recompose)."""
        return capi.recompose(self.FK.detach(), self.FC.detach(), self.FH.detach(),
                              self.FW.detach())


class CP3Conv2dFunction(torch.autograd.Function):
    """The 3-factor CP convolution of the reference's ``Conv2dCpFusedNchw`` op
    (Kernels/cp_fused_nchw.cc:6-30; its Python definition is pointwise K0,
    depthwise K1, pointwise K2, test/layers.py:265-282):

        y[n,t] = sum_r K2[r,t] * (K1[:,:,r] (*) sum_c K0[c,r] x[n,c])

    K0 [C,R], K1 [Y,X,R], K2 [R,T].  All three passes are the library's cp3 entry
    points.
    """

    @staticmethod
    def forward(ctx, x, K0, K1, K2, pad):
        if 2 * pad + 1 != K1.shape[0] or 2 * pad + 1 != K1.shape[1]:
            raise ValueError("autograd binding needs 2*pad = Y-1 = X-1")
        K0, K1, K2 = (t.contiguous().float() for t in (K0, K1, K2))
        x = x.contiguous().float()
        ctx.pad = pad
        ctx.save_for_backward(x, K0, K1, K2)
        return capi.cp3_conv2d_forward(x, K0, K1, K2, pad=pad)

    @staticmethod
    def backward(ctx, dy):
        x, K0, K1, K2 = ctx.saved_tensors
        dy = dy.contiguous().float()
        dx = None
        if ctx.needs_input_grad[0]:
            dx = capi.cp3_conv2d_backward_data(dy, K0, K1, K2, pad=ctx.pad)
        grads = (None, None, None)
        if any(ctx.needs_input_grad[1:4]):
            grads = capi.cp3_conv2d_backward_filter(x, dy, K0, K1, K2, pad=ctx.pad)
            grads = tuple(g if need else None for g, need in zip(grads, ctx.needs_input_grad[1:4]))
        _after_backward()
        return (dx,) + grads + (None,)


def cp3_conv2d(x, K0, K1, K2, pad):
    """Functional form of the differentiable 3-factor CP convolution (NCHW)."""
    return CP3Conv2dFunction.apply(x, K0, K1, K2, pad)


class CP3Conv2d(torch.nn.Module):
    """A rank-R 3-factor CP convolution layer, "same" padding: pointwise K0 [C,R],
    depthwise K1 [k,k,R], pointwise K2 [R,T] (the kernels of the reference's Python
    layer, test/layers.py:285-294, in the fused op's layouts).  Factors start as
    normal(0, s) with s chosen so that the equivalent dense filter
    sum_r K0[c,r] K1[i,j,r] K2[r,t] has the variance of a Kaiming-normal one."""

    def __init__(self, in_channels, out_channels, kernel_size, rank, device="cuda"):
        super().__init__()
        if kernel_size % 2 != 1:
            raise ValueError("kernel_size must be odd (same padding)")
        self.pad = kernel_size // 2
        fan_in = in_channels * kernel_size * kernel_size
        # Var = R * s^6 for three independent N(0, s^2) factors; target 2 / fan_in
        s = (2.0 / (fan_in * rank)) ** (1.0 / 6.0)
        mk = lambda *d: torch.nn.Parameter(torch.randn(*d, device=device) * s)
        self.K0 = mk(in_channels, rank)
        self.K1 = mk(kernel_size, kernel_size, rank)
        self.K2 = mk(rank, out_channels)

    def forward(self, x):
        return cp3_conv2d(x, self.K0, self.K1, self.K2, self.pad)


class RCPConv2dFunction(torch.autograd.Function):
    """The reshaped-CP convolution of the reference's ``Conv2dRcpFusedNchw`` op
    (Kernels/rcp_fused_nchw.cc:6-12; test/test_conv2d_rcp.py:38-41):

        y[n,(x,y)] = sum_r sum_{a,b} K0[a,x,r] K1[b,y,r] * (KC[:,:,r] (*) x[n,(a,b)])

    K0 [S0,T0,R], K1 [S1,T1,R], KC [Y,X,R]; x has S0*S1 channels, y T0*T1.  All three
    passes are the library's rcp entry points."""

    @staticmethod
    def forward(ctx, x, K0, K1, KC, pad):
        if 2 * pad + 1 != KC.shape[0] or 2 * pad + 1 != KC.shape[1]:
            raise ValueError("autograd binding needs 2*pad = Y-1 = X-1")
        K0, K1, KC = (t.contiguous().float() for t in (K0, K1, KC))
        x = x.contiguous().float()
        ctx.pad = pad
        ctx.save_for_backward(x, K0, K1, KC)
        return capi.rcp_conv2d_forward(x, K0, K1, KC, pad=pad)

    @staticmethod
    def backward(ctx, dy):
        x, K0, K1, KC = ctx.saved_tensors
        dy = dy.contiguous().float()
        dx = None
        if ctx.needs_input_grad[0]:
            dx = capi.rcp_conv2d_backward_data(dy, K0, K1, KC, pad=ctx.pad)
        grads = (None, None, None)
        if any(ctx.needs_input_grad[1:4]):
            grads = capi.rcp_conv2d_backward_filter(x, dy, K0, K1, KC, pad=ctx.pad)
            grads = tuple(g if need else None for g, need in zip(grads, ctx.needs_input_grad[1:4]))
        _after_backward()
        return (dx,) + grads + (None,)


def rcp_conv2d(x, K0, K1, KC, pad):
    """Functional form of the differentiable reshaped-CP convolution (NCHW)."""
    return RCPConv2dFunction.apply(x, K0, K1, KC, pad)


class AdapterLinearFunction(torch.autograd.Function):
    """``adapter_linear`` as a Python autograd function: stands for the native one
    (csrc/torch/binding.cpp) where a call has to be seen as an operator, in a trace."""

    @staticmethod
    def forward(ctx, x, W, A, B, ids, scale=None, bias=None, scales=None, features=None):
        """``scales``: of W, whose codes are in its place then (an argument each, so that a trace sees both), of
        ``features`` values a row."""
        need = ctx.needs_input_grad
        ctx.codes, ctx.features = scales is not None, features
        if scales is not None:
            W = capi.Mx4(W, scales, features)
        rows = (W.codes if scales is not None else W).shape[:1]
        if need[1] or need[5] or need[6]:
            raise ValueError("the projection, its bias and the scales are not trained: detach them")
        factors = need[2] or need[3]
        # (made by an operator, or the trace would not know it)
        y = torch.empty(x.shape[:-1] + rows, dtype=x.dtype, device=x.device)
        kept = None
        if factors:
            _, kept = capi.adapter_forward(x, W, A, B, ids, scale, bias, out=y, keep=True)
        else:
            capi.adapter_forward(x, W, A, B, ids, scale, bias, out=y)
        ctx.save_for_backward(x if factors else None, W.codes if ctx.codes else W, A, B, ids, scale, kept, scales)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, W, A, B, ids, scale, kept, scales = ctx.saved_tensors
        if ctx.codes:
            W = capi.Mx4(W, scales, ctx.features)
        need = ctx.needs_input_grad
        dx, dA, dB = capi.adapter_backward(dy.to(A.dtype), x, W, A, B, ids, scale, kept, want_dx=need[0],
                                           want_factors=need[2] or need[3])
        if torch.is_grad_enabled():              # (create_graph: as the native one)
            told = torch._C._functions.DelayedError(b"the gradients of adapter_linear cannot be differentiated again", 1)
            dx, dA, dB = (g if g is None else told(g.detach().requires_grad_()) for g in (dx, dA, dB))
        return dx, None, dA if need[2] else None, dB if need[3] else None, None, None, None, None, None


def adapter_linear(x, W, A, B, ids, scale=None, bias=None):
    """Functional form of a dense projection with the low-rank adapters of many requests
    beside it (``capi.adapter_forward``), differentiable in x, A and B.

    W may be held in 4 bits (``capi.Mx4``).  W and bias are frozen: a call that asks for their gradient raises ``ValueError``.  The gradients themselves
    are not differentiable: after ``create_graph=True`` a second derivative raises."""
    # torch.jit.trace records operators: the native call would leave a constant in the graph
    if torch._C._get_tracing_state() is None:
        return capi._native.adapter_linear(x, W, A, B, ids, scale, bias)
    codes, scales = (W.codes, W.scales) if isinstance(W, capi.Mx4) else (W, None)
    return AdapterLinearFunction.apply(x, codes, A, B, ids, scale, bias, scales, W.features if scales is not None else None)


class AdapterLinear(torch.nn.Module):
    """A frozen dense projection [out_features, in_features] with ``adapters`` low-rank
    adapters of rank ``rank`` that are trained, each token through the one that ``ids`` names.

    A starts as normal(0, 1 / sqrt(in_features)), B as zero, so that an adapter starts as
    nothing; ``alpha / rank`` scales all of them.  ``weight`` and ``bias``: the projection's, as of
    a trained layer (kept as buffers); without them it starts as a Kaiming-normal one.  ``.to(dtype)``, ``.half()``
    and ``.bfloat16()`` convert the projection and the adapters; scales and bias stay float32.  ``weight_bits=4``: the
    projection is held in microscaled 4-bit floating point (``weight_codes`` and ``weight_scales``, 17 / 32 of a byte a value)."""

    weight_bits = None

    def __init__(self, in_features, out_features, rank, adapters=1, alpha=None, weight=None, bias=None,
                 dtype=torch.float32, device="cuda", weight_bits=None):
        super().__init__()
        if weight is None:
            weight = torch.randn(out_features, in_features, device=device) * (2.0 / in_features) ** 0.5
        if tuple(weight.shape) != (out_features, in_features):
            raise ValueError("weight must be [out_features, in_features]")
        if weight_bits not in (None, 4):
            raise ValueError("weight_bits must be None or 4")
        self.weight_bits = weight_bits
        if weight_bits is None:
            self.register_buffer("weight", weight.detach().to(device, dtype))
        else:
            q = capi.mx4_quantize(weight.detach().to(device))
            self.register_buffer("weight_codes", q.codes)
            self.register_buffer("weight_scales", q.scales)
        self.register_buffer("bias", None if bias is None else bias.detach().to(device, torch.float32))
        self.register_buffer("scale", torch.full((adapters,), (rank if alpha is None else alpha) / rank,
                                                 dtype=torch.float32, device=device))
        self.A = torch.nn.Parameter((torch.randn(adapters, rank, in_features, device=device) *
                                     in_features ** -0.5).to(dtype))
        self.B = torch.nn.Parameter(torch.zeros(adapters, out_features, rank, device=device, dtype=dtype))

    def _apply(self, fn, recurse=True):
        """Conversions of a network leave the scales and the bias what they are, float32, as the layer takes them."""
        before = {k: self._buffers[k] for k in ("scale", "bias")}
        super()._apply(fn, recurse)
        for k, old in before.items():
            new = self._buffers[k]
            if new is not None and new.dtype != torch.float32:
                self._buffers[k] = old.to(new.device, torch.float32)
        return self

    def projection(self):
        """The projection as ``capi.adapter_forward`` takes it: ``weight``, or a ``capi.Mx4``."""
        return self.weight if self.weight_bits is None else capi.Mx4(self.weight_codes, self.weight_scales, self.A.shape[-1])

    def forward(self, x, ids):
        return adapter_linear(x, self.projection(), self.A, self.B, ids, self.scale, self.bias)


_NO_GRADIENT = "activations in 4 bits have no gradient: detach them, or call without gradients"


class Mx4LinearFunction(torch.autograd.Function):
    """``mx4_linear`` as a Python autograd function: stands for the native one (csrc/torch/binding.cpp) where a
    call has to be seen as an operator, in a trace.  ``activations``: as ``capi.mx4_linear`` takes it."""

    @staticmethod
    def forward(ctx, x, codes, scales, bias, features, activations=None):
        if ctx.needs_input_grad[3]:
            raise ValueError("the projection and its bias are not trained: detach them")
        y = torch.empty(x.shape[:-1] + codes.shape[:1], dtype=x.dtype, device=x.device)   # (made by an operator)
        capi.mx4_linear(x, capi.Mx4(codes, scales, features), bias, activations, out=y)
        ctx.save_for_backward(codes, scales)
        ctx.features, ctx.dtype, ctx.activations = features, x.dtype, activations
        return y

    @staticmethod
    def backward(ctx, dy):
        codes, scales = ctx.saved_tensors
        if ctx.activations is not None:
            raise ValueError(_NO_GRADIENT)
        dx = capi.mx4_linear_backward(dy.detach().to(ctx.dtype), capi.Mx4(codes, scales, ctx.features))
        if torch.is_grad_enabled() and dy.requires_grad:             # (create_graph: as the native one)
            told = torch._C._functions.DelayedError(b"the gradients of mx4_linear cannot be differentiated again", 1)
            dx = told(dx.requires_grad_())
        return dx, None, None, None, None, None


def mx4_linear(x, W, bias=None):
    """Functional form of a dense projection whose weights are held in 4 bits (``capi.mx4_linear``), differentiable
    in x.  W and bias are frozen: a call that asks for the bias's gradient raises ``ValueError``."""
    if torch._C._get_tracing_state() is None:
        return capi._native.mx4_linear_grad(x, W, bias)
    return Mx4LinearFunction.apply(x, W.codes, W.scales, bias, W.features)


class Mx4Linear(torch.nn.Module):
    """A frozen dense projection held in microscaled 4-bit floating point.  ``weight`` [out_features, in_features] and
    ``bias``: of a trained layer.  ``activations=4``: inputs are rounded to 4 bits as well; such a layer has no gradients."""

    def __init__(self, weight, bias=None, activations=None, device="cuda"):
        super().__init__()
        if activations not in (None, 4):
            raise ValueError("activations must be None or 4")
        self.in_features, self.activations = weight.shape[1], activations
        q = capi.mx4_quantize(weight.detach().to(device))
        self.register_buffer("weight_codes", q.codes)
        self.register_buffer("weight_scales", q.scales)
        self.register_buffer("bias", None if bias is None else bias.detach().to(device, torch.float32))

    def _apply(self, fn, recurse=True):
        """Conversions of a network leave the bias float32."""
        old = self.bias
        super()._apply(fn, recurse)
        if old is not None and self.bias.dtype != torch.float32:
            self.bias = old.to(self.bias.device, torch.float32)
        return self

    def forward(self, x):
        W = capi.Mx4(self.weight_codes, self.weight_scales, self.in_features)
        if self.activations is None:
            return mx4_linear(x, W, self.bias)
        if torch.is_grad_enabled() and x.requires_grad:
            raise ValueError(_NO_GRADIENT)
        if torch._C._get_tracing_state() is not None:
            return Mx4LinearFunction.apply(x, W.codes, W.scales, self.bias, W.features, self.activations)
        return capi.mx4_linear(x, W, self.bias, activations=4)


class LayerNormFunction(torch.autograd.Function):
    """``layer_norm`` as a Python autograd function: stands for the native one (csrc/torch/binding.cpp) where a
    call has to be seen as an operator, in a trace."""

    @staticmethod
    def forward(ctx, x, weight=None, bias=None, eps=1e-5):
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)     # (made by an operator, or the trace would not know it)
        _, stats = capi.layer_norm_forward(x, weight, bias, eps, out=y, keep=True)
        ctx.save_for_backward(x, weight, stats)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        grads = capi.layer_norm_backward(dy.to(x.dtype), x, weight, stats, *ctx.needs_input_grad[:3])
        if torch.is_grad_enabled():              # (create_graph: as the native one)
            told = torch._C._functions.DelayedError(b"the gradients of layer_norm cannot be differentiated again", 1)
            grads = tuple(g if g is None else told(g.detach().requires_grad_()) for g in grads)
        return *grads, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Functional form of the layer norm over x's last dimension (``capi.layer_norm_forward``), differentiable in
    x, weight and bias.  The gradients themselves are not differentiable."""
    # torch.jit.trace records operators: the native call would leave a constant in the graph
    if torch._C._get_tracing_state() is None:
        return capi._native.layer_norm(x, weight, bias, eps)
    return LayerNormFunction.apply(x, weight, bias, eps)


class LayerNorm(torch.nn.Module):
    """Layer norm over the last dimension of ``features`` values, with a weight and (``bias``) a bias that start as
    1 and 0.  ``.to(dtype)``, ``.half()`` and ``.bfloat16()`` of a network leave both float32, as the layer takes them:
    its output is of its input's type."""

    def __init__(self, features, eps=1e-5, bias=True, device="cuda"):
        super().__init__()
        self.eps = eps
        self.weight = torch.nn.Parameter(torch.ones(features, device=device))
        self.bias = torch.nn.Parameter(torch.zeros(features, device=device)) if bias else None

    def _apply(self, fn, recurse=True):
        """Conversions of a network leave weight and bias float32."""
        def kept(t):
            new = fn(t)
            return new if new.dtype == torch.float32 else t.to(new.device)
        return super()._apply(kept, recurse)

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias, self.eps)
