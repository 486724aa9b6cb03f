"""Microscaled 4-bit floating point: rounding, reading back, and projections whose weights are held in it, against their
definition in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
LEVELS = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


@pytest.fixture(scope="module")
def cp4():
    import paralleltnnlayers_amd as cp4
    cp4.lib()
    return cp4


def rounded(x):
    """(codes, scales, values) of rows, in 64 bits on the CPU."""
    x = x.double().cpu()
    rows, K = x.shape
    blocks = -(-K // 32)
    v = torch.nn.functional.pad(x, (0, blocks * 32 - K)).view(rows, blocks, 32)
    top = v.abs().amax(2)
    good = top < math.inf
    e = torch.frexp(torch.where(good, top, torch.ones_like(top))).exponent - 3
    e = torch.where(top > 0, e, torch.full_like(e, -127)).clamp(min=-127)
    v = torch.where(good[..., None], v, torch.zeros_like(v)) / torch.exp2(e.double())[..., None]
    d = (v.abs()[..., None] - LEVELS).abs()
    near = d == d.amin(-1, keepdim=True)                             # (two at a tie: the even one)
    even = near & (torch.arange(8) % 2 == 0)
    q = torch.where(even.any(-1), even.double().argmax(-1), near.double().argmax(-1))
    values = LEVELS[q] * v.sign() * torch.exp2(e.double())[..., None]
    values = torch.where(good[..., None], values, torch.full_like(values, math.nan))
    q = q + 8 * (torch.signbit(v) & good[..., None])
    scales = torch.where(good, e + 127, torch.full_like(e, 255)).to(torch.uint8)
    codes = (q[..., 0::2] | q[..., 1::2] << 4).to(torch.uint8).view(rows, blocks * 16)
    return codes, scales, values.view(rows, -1)[:, :K]


def same(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(7.0, 8.0, 9.0), b.nan_to_num(7.0, 8.0, 9.0))


def make(*shape, dtype=torch.float32, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * torch.randn(shape[-1], generator=g).exp() * std).to(dtype).cuda()


# ---- rounding ----------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", list(DTYPES), ids=str)
@pytest.mark.parametrize("shape", [(1, 1), (1, 31), (3, 32), (5, 33), (7, 64), (2, 1000), (33, 1001), (300, 260), (1, 25088), (4097, 40)], ids=str)
def test_rounding(cp4, shape, dtype):
    x = make(*shape, dtype=DTYPES[dtype])
    q = cp4.mx4_quantize(x)
    codes, scales, values = rounded(x)
    assert q.features == shape[1] and torch.equal(q.codes.cpu(), codes) and torch.equal(q.scales.cpu(), scales)
    for t in DTYPES.values():
        y = cp4.mx4_dequantize(q, t)
        assert y.dtype == t and torch.equal(y.double().cpu(), values.to(t).double())


def test_ties_ends_and_tiny_values(cp4):
    edges = (LEVELS[1:] + LEVELS[:-1]) / 2
    near = torch.cat([edges, edges * (1 - 2.0 ** -23), edges * (1 + 2.0 ** -22), LEVELS, torch.tensor([7.0, 7.999])])
    near = torch.cat([near, -near]).float()
    rows = []
    for e in (-126, -125, -124, -60, 0, 60, 120):
        for i in range(0, len(near), 31):                            # (a 6 in each block, so that its scale is known)
            rows.append(torch.cat([torch.tensor([6.0]), near[i:i + 31], torch.zeros(31)])[:32].double() * 2.0 ** e)
    rows.append(torch.full((32,), 2.0 ** -149).double())             # the smallest values, zeros, and the largest
    rows.append(torch.tensor([2.0 ** -149, -2.0 ** -130, 2.0 ** -127, 3 * 2.0 ** -128] * 8).double())
    rows.append(torch.tensor([0.0, -0.0] * 16).double())
    rows.append(torch.tensor([torch.finfo(torch.float32).max, -1e38] * 16).double())
    x = torch.stack(rows).float().cuda()
    q = cp4.mx4_quantize(x)
    codes, scales, values = rounded(x)
    assert torch.equal(q.scales.cpu(), scales) and torch.equal(q.codes.cpu(), codes)
    assert torch.equal(cp4.mx4_dequantize(q).double().cpu(), values.float().double())


@pytest.mark.parametrize("dtype", list(DTYPES), ids=str)
def test_blocks_that_are_not_finite(cp4, dtype):
    x = make(6, 100, dtype=DTYPES[dtype])
    x[0, 3], x[1, 40], x[2, 99], x[3, 64] = math.inf, -math.inf, math.nan, math.nan
    q = cp4.mx4_quantize(x)
    codes, scales, values = rounded(x)
    assert torch.equal(q.codes.cpu(), codes) and torch.equal(q.scales.cpu(), scales)
    for t in DTYPES.values():
        assert same(cp4.mx4_dequantize(q, t), values)


def test_every_code_and_scale_reads_back(cp4):
    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1)      # 512 values a row, of one scale
    scales = torch.arange(256, dtype=torch.uint8)[:, None].repeat(1, 16)
    q = cp4.Mx4(codes.cuda(), scales.cuda(), 512)
    code = torch.stack([codes & 15, codes >> 4], 2).view(256, 512).long()
    want = LEVELS[code & 7] * torch.where(code > 7, -1.0, 1.0).double() * torch.exp2(scales.double() - 127).repeat_interleave(32, 1)
    want[255] = math.nan
    for t in DTYPES.values():
        assert same(cp4.mx4_dequantize(q, t), want.float().to(t))


def test_strides_dimensions_and_no_rows(cp4):
    x = make(24, 100, dtype=torch.bfloat16)
    q = cp4.mx4_quantize(x)
    wide = torch.zeros(24, 333, dtype=x.dtype, device="cuda")
    wide[:, 7:107] = x
    for view in (wide[:, 7:107], x.t().contiguous().t(), x.view(2, 3, 4, 100)):
        r = cp4.mx4_quantize(view)
        assert torch.equal(r.codes.view(24, -1), q.codes) and torch.equal(r.scales.view(24, -1), q.scales)
        assert cp4.mx4_dequantize(r, torch.float32).shape == view.shape
    empty = cp4.mx4_quantize(x[:0])
    assert empty.codes.shape == (0, 64) and cp4.mx4_dequantize(empty).shape == (0, 100)
    out = torch.zeros(24, 100, dtype=torch.float16, device="cuda")
    assert cp4.mx4_dequantize(q, out=out) is out and same(out, cp4.mx4_dequantize(q, torch.float16))


# ---- projections ---------------------------------------------------------------------------------------

def bound(want, size, dtype, terms):
    """Half a step of the type, and fp32 sums of `terms` products in any order that adds up at least eight at a time."""
    b = want.abs() * torch.finfo(dtype).eps / 2 + size * 2.0 ** -24 * (terms / 8 + 64)
    return b + 2.0 ** -25 if dtype == torch.float16 else b


def close(got, want, size, dtype, terms):
    assert got.dtype == dtype and got.shape == want.shape
    off, most = (got.double().cpu() - want).abs(), bound(want, size, dtype, terms)
    assert (off <= most).all(), float((off / most).nan_to_num().max())


def weights(cp4, N, K, dtype, seed=1):
    """W in 4 bits, and its values in 64 bits as x's type holds them."""
    q = cp4.mx4_quantize(make(N, K, seed=seed, std=K ** -0.5))
    return q, rounded_values(cp4, q, dtype)


def rounded_values(cp4, q, dtype):
    return cp4.mx4_dequantize(q, dtype).double().cpu()


LINEAR = [(1, 1, 1), (1, 1024, 1024), (2, 33, 17), (3, 130, 64), (5, 257, 100), (16, 4096, 80), (17, 1000, 333), (31, 96, 200), (33, 500, 48),
          (48, 640, 1000), (64, 1001, 130), (65, 1001, 130), (100, 64, 64), (130, 777, 300), (257, 96, 1100), (333, 1001, 777),
          (700, 320, 520), (1031, 200, 260), (300, 4100, 96)]


@pytest.mark.parametrize("dtype", list(DTYPES), ids=str)
@pytest.mark.parametrize("T,K,N", LINEAR)
def test_linear(cp4, T, K, N, dtype):
    t = DTYPES[dtype]
    q, W = weights(cp4, N, K, t)
    x, bias = make(T, K, dtype=t), make(N)
    X = x.double().cpu()
    for b in (None, bias):
        want, size = X @ W.T, X.abs() @ W.abs().T
        if b is not None:
            want, size = want + b.double().cpu(), size + b.double().cpu().abs()
        close(cp4.mx4_linear(x, q, b), want, size, t, K)
    dy = make(T, N, dtype=t, seed=5)
    D = dy.double().cpu()
    close(cp4.mx4_linear_backward(dy, q), D @ W, D.abs() @ W.abs(), t, N)


@pytest.mark.parametrize("dtype", list(DTYPES), ids=str)
@pytest.mark.parametrize("T,K,N", LINEAR + [(600, 2100, 520)])
def test_both_operands_in_4_bits(cp4, T, K, N, dtype):
    t = DTYPES[dtype]
    q = cp4.mx4_quantize(make(N, K, seed=1, std=K ** -0.5))
    x, bias = make(T, K, dtype=t), make(N)
    X, W = rounded(x)[2], cp4.mx4_dequantize(q).double().cpu()
    want, size = X @ W.T, X.abs() @ W.abs().T
    close(cp4.mx4_linear(x, q, activations=4), want, size, t, K)
    bd = bias.double().cpu()
    xq = cp4.mx4_quantize(x)
    y = cp4.mx4_linear(xq, q, bias, dtype=t)
    close(y, want + bd, size + bd.abs(), t, K)
    assert torch.equal(y, cp4.mx4_linear(x, q, bias, activations=4))


@pytest.mark.parametrize("dtype", list(DTYPES), ids=str)
@pytest.mark.parametrize("T", [2, 16, 17, 32, 33, 48, 49, 64])
def test_few_rows(cp4, T, dtype):
    """Depths from less than a wave's turn to several of each wave, with and without a rest, rows on 16-byte boundaries and off them."""
    for K, N in ((104, 40), (640, 33), (1024, 300), (3200, 70), (4200, 2000)):
        q, W = weights(cp4, N, K, DTYPES[dtype])
        x = make(T, K, dtype=DTYPES[dtype])
        X = x.double().cpu()
        for rows in (x, torch.cat([x, x[:, :1]], 1)[:, :K]):
            close(cp4.mx4_linear(rows, q), X @ W.T, X.abs() @ W.abs().T, DTYPES[dtype], K)


@pytest.mark.parametrize("T, ld", [(5, 1 << 29), (40, 1 << 27), (300, 1 << 24)])
def test_rows_beyond_32_bit_offsets(cp4, T, ld):
    K, N = 264, 200
    q, W = weights(cp4, N, K, torch.bfloat16)
    x, dy = make(T, K, dtype=torch.bfloat16), make(T, N, dtype=torch.bfloat16, seed=3)
    room = torch.empty((T - 1) * ld + 512, dtype=torch.bfloat16, device="cuda")
    assert room.numel() * 2 > 1 << 32
    wide = room.as_strided((T, K), (ld, 1))
    wide.copy_(x)
    X, D = x.double().cpu(), dy.double().cpu()
    close(cp4.mx4_linear(wide, q), X @ W.T, X.abs() @ W.abs().T, torch.bfloat16, K)
    four, want = cp4.mx4_quantize(wide), cp4.mx4_quantize(x)
    assert torch.equal(four.codes, want.codes) and torch.equal(four.scales, want.scales)
    wide = room.as_strided((T, N), (ld, 1))
    wide.copy_(dy)
    close(cp4.mx4_linear_backward(wide, q), D @ W, D.abs() @ W.abs(), torch.bfloat16, N)


def test_codes_beyond_32_bit_offsets(cp4):
    """W of more than 4 GiB of codes, read by the kernels of few and of many rows, as values and as codes, both ways.  x has 16 values a
    row, so that sums are short; of dx some columns are looked at."""
    K, N = 1 << 22, 2100
    W = torch.empty(N, K, dtype=torch.bfloat16, device="cuda")
    for n in range(0, N, 300):
        W[n:n + 300].normal_(generator=torch.Generator("cuda").manual_seed(n))
    q = cp4.mx4_quantize(W)
    assert q.codes.numel() > 1 << 32
    cp4.mx4_dequantize(q, torch.bfloat16, out=W)
    at = torch.tensor([0, 1, 33, 4095, K // 2 + 5, K - 64, K - 2, K - 1] + [K // 9 * k for k in range(1, 9)])
    V = W[:, at.cuda()].double().cpu()
    for n in (0, 1023, N - 1):
        assert same(W[n], cp4.mx4_dequantize(cp4.Mx4(q.codes[n:n + 1], q.scales[n:n + 1], K), torch.bfloat16)[0])
    del W
    for T in (3, 60, 100):
        x = torch.zeros(T, K, dtype=torch.bfloat16, device="cuda")
        X = make(T, 16, dtype=torch.bfloat16, seed=T)
        x[:, at.cuda()] = X
        X = X.double().cpu()
        close(cp4.mx4_linear(x, q), X @ V.T, X.abs() @ V.abs().T, torch.bfloat16, 16)
        four = cp4.mx4_quantize(x)
        R = cp4.mx4_dequantize(four, torch.bfloat16)[:, at.cuda()].double().cpu()
        close(cp4.mx4_linear(four, q, dtype=torch.bfloat16), R @ V.T, R.abs() @ V.abs().T, torch.bfloat16, 16)
        dy = make(T, N, dtype=torch.bfloat16, seed=T + 1)
        D = dy.double().cpu()
        close(cp4.mx4_linear_backward(dy, q)[:, at.cuda()], D @ V, D.abs() @ V.abs(), torch.bfloat16, N)


def test_large_results(cp4):
    """Results that go past the caches are the same ones."""
    K = (1 << 22) - 3
    x = make(30, K, dtype=torch.bfloat16)
    q = cp4.mx4_quantize(x)
    y = cp4.mx4_dequantize(q, torch.bfloat16)
    assert y.numel() * 2 >= 224 << 20
    for t in (0, 13, 29):
        row = cp4.mx4_quantize(x[t:t + 1])
        assert torch.equal(q.codes[t:t + 1], row.codes) and torch.equal(y[t:t + 1], cp4.mx4_dequantize(row, torch.bfloat16))


def test_large_tiles(cp4):
    """Shapes that every tile has whole ones and edges of."""
    T, K, N = 2100, 1060, 2060
    q, W = weights(cp4, N, K, torch.bfloat16)
    x, dy = make(T, K, dtype=torch.bfloat16), make(T, N, dtype=torch.bfloat16, seed=3)
    X, D = x.double().cpu(), dy.double().cpu()
    close(cp4.mx4_linear(x, q), X @ W.T, X.abs() @ W.abs().T, torch.bfloat16, K)
    close(cp4.mx4_linear_backward(dy, q), D @ W, D.abs() @ W.abs(), torch.bfloat16, N)
    R = rounded(x)[2]
    close(cp4.mx4_linear(x, q, activations=4), R @ W.T, R.abs() @ W.abs().T, torch.bfloat16, K)


@pytest.mark.parametrize("dtype", list(DTYPES), ids=str)
@pytest.mark.parametrize("T", [1, 13, 70, 300])
def test_strides_of_activations(cp4, T, dtype):
    t = DTYPES[dtype]
    q, _ = weights(cp4, 100, 333, t)
    x, dy = make(T, 333, dtype=t), make(T, 100, dtype=t, seed=2)
    wide = torch.zeros(T, 1001, dtype=t, device="cuda")
    wx, wdy = wide[:, 5:338], wide[:, 401:501]
    wx.copy_(x)
    wdy.copy_(dy)
    assert torch.equal(cp4.mx4_linear(wx, q), cp4.mx4_linear(x, q))
    assert torch.equal(cp4.mx4_linear(wx, q, activations=4), cp4.mx4_linear(x, q, activations=4))
    assert torch.equal(cp4.mx4_linear_backward(wdy, q), cp4.mx4_linear_backward(dy, q))
    out = torch.zeros(T, 100, dtype=t, device="cuda")
    assert cp4.mx4_linear(x, q, out=out) is out and torch.equal(out, cp4.mx4_linear(x, q))
    shifted = torch.empty(q.codes.numel() + 1, dtype=torch.uint8, device="cuda")[1:].view_as(q.codes).copy_(q.codes)
    assert torch.equal(cp4.mx4_linear(x, cp4.Mx4(shifted, q.scales, 333)), out)
    assert cp4.mx4_linear(x[:0], q).shape == (0, 100) and cp4.mx4_linear(x[:0], q, activations=4).shape == (0, 100)
    assert cp4.mx4_linear_backward(dy[:0], q).shape == (0, 333)
    assert torch.equal(cp4.mx4_linear(x.view(1, T, 333), q)[0], out)


@pytest.mark.parametrize("T", [3, 90, 300])
def test_what_is_not_finite_stays_with_its_row(cp4, T):
    """A token's infinity or NaN in its row of y, a NaN block of W in its output."""
    x = make(T, 200, dtype=torch.bfloat16)
    W = make(70, 200, seed=1)
    for four in (None, 4):
        clean = cp4.mx4_linear(x, cp4.mx4_quantize(W), activations=four)
        bx, bW = x.clone(), W.clone()
        bx[1, 150], bx[2, 3] = math.inf, math.nan
        bW[5, 199] = math.nan
        y = cp4.mx4_linear(bx, cp4.mx4_quantize(bW), activations=four)
        bad = torch.zeros(T, 70, dtype=torch.bool)
        bad[1:3] = bad[:, 5] = True
        assert not y[bad.cuda()].isfinite().any()
        assert torch.equal(y[~bad.cuda()], clean[~bad.cuda()])


@pytest.mark.parametrize("dtype", list(DTYPES), ids=str)
@pytest.mark.parametrize("T,K,N,R,G", [(1, 64, 48, 4, 2), (7, 1001, 130, 5, 3), (40, 512, 256, 16, 40), (64, 130, 65, 33, 5), (90, 320, 200, 8, 4),
                                       (60, 1040, 48, 200, 3), (64, 1040, 48, 100, 6), (30, 2048, 300, 256, 2), (300, 1001, 130, 7, 5), (700, 256, 600, 64, 3)])
def test_adapters(cp4, T, K, N, R, G, dtype):
    """The adapters beside a projection in 4 bits are those beside one of its values."""
    t = DTYPES[dtype]
    q, W = weights(cp4, N, K, t)
    x, A, B = make(T, K, dtype=t), make(G, R, K, dtype=t, seed=2, std=K ** -0.5), make(G, N, R, dtype=t, seed=3)
    g = torch.Generator().manual_seed(4)
    ids = torch.randint(-1, G, (T,), generator=g).int().cuda()
    scale, bias, dy = torch.rand(G, generator=g).cuda(), make(N, seed=6), make(T, N, dtype=t, seed=7)
    y, kept = cp4.adapter_forward(x, q, A, B, ids, scale, bias, keep=True)
    grads = cp4.adapter_backward(dy, x, q, A, B, ids, scale, kept)
    # in 64 bits
    X, D, i = x.double().cpu(), dy.double().cpu(), ids.cpu().long()
    own, s = i >= 0, scale.double().cpu()[i.clamp(min=0)] * (i >= 0)
    At, Bt = A.double().cpu()[i.clamp(min=0)], B.double().cpu()[i.clamp(min=0)]
    h = torch.einsum("trk,tk->tr", At, X) * s[:, None]
    dh = torch.einsum("tnr,tn->tr", Bt, D) * s[:, None]
    # (h has 16 bits behind it where the type has 16: 2^-16 of each rank's size)
    off = 2.0 ** -16 if t != torch.float32 else 2.0 ** -22
    h_size = torch.einsum("trk,tk->tr", At.abs(), X.abs()) * s[:, None]
    dh_size = torch.einsum("tnr,tn->tr", Bt.abs(), D.abs()) * s[:, None]
    want = X @ W.T + bias.double().cpu() + torch.einsum("tnr,tr->tn", Bt, h)
    more = torch.einsum("tnr,tr->tn", Bt.abs(), h_size)
    size = X.abs() @ W.abs().T + bias.double().cpu().abs() + more * (1 + off * 2.0 ** 24 / (K / 8 + 64))
    close(y, want, size, t, K)
    want = D @ W + torch.einsum("trk,tr->tk", At, dh)
    size = D.abs() @ W.abs() + torch.einsum("trk,tr->tk", At.abs(), dh_size) * (1 + off * 2.0 ** 24 / (N / 8 + 64))
    close(grads[0], want, size, t, N)
    # the adapters' gradients do not see W
    plain = cp4.adapter_backward(dy, x, W.to(t).cuda(), A, B, ids, scale, kept)
    assert torch.equal(grads[1], plain[1]) and torch.equal(grads[2], plain[2])
    assert own.any() or T == 1


def test_module_training_and_trace(cp4):
    """A layer held in 4 bits is the layer of its values: output, gradients, converted, traced, saved."""
    from paralleltnnlayers_amd import torch_ops
    torch.manual_seed(0)
    W, bias = torch.randn(48, 70), torch.randn(48)
    four = torch_ops.AdapterLinear(70, 48, 8, adapters=3, weight=W, bias=bias, weight_bits=4)
    q = cp4.Mx4(four.weight_codes, four.weight_scales, 70)
    plain = torch_ops.AdapterLinear(70, 48, 8, adapters=3, weight=cp4.mx4_dequantize(q), bias=bias)
    with torch.no_grad():
        four.B.copy_(torch.randn(four.B.shape))
        plain.A.copy_(four.A)
        plain.B.copy_(four.B)
    ids = torch.tensor([0, 1, 2, -1, 2, 2, 1, 0, 0, 1] * 30, device="cuda", dtype=torch.int32)
    for dtype in (torch.float32, torch.bfloat16):
        four.to(dtype)
        plain.to(dtype)
        assert four.weight_codes.dtype == torch.uint8 and four.bias.dtype == torch.float32
        x, dy = torch.randn(300, 70, device="cuda").to(dtype), torch.randn(300, 48, device="cuda").to(dtype)
        results = []
        for run in (four, plain, torch.jit.trace(four, (x[:20], ids[:20]), check_trace=False)):
            leaf = x.clone().requires_grad_()
            y = run(leaf, ids)
            results.append([y.detach(), *torch.autograd.grad(y, [leaf, (four if run is not plain else plain).A, (four if run is not plain else plain).B], dy)])
        for a, b, c in zip(*results):
            step = torch.finfo(dtype).eps
            # (the order of a sum differs: a rounding more or less, and fp32 sums of 70)
            assert (a - b).abs().max() <= 2 * step * b.abs().max() and torch.equal(a, c)
    again = torch_ops.AdapterLinear(70, 48, 8, adapters=3, bias=torch.zeros(48), weight_bits=4, dtype=torch.bfloat16)
    again.load_state_dict(four.state_dict())
    assert torch.equal(again(x, ids), four(x, ids))

    dense = torch_ops.Mx4Linear(W, bias)
    leaf = x.float().requires_grad_()
    y = dense(leaf)
    (dx,) = torch.autograd.grad(y, [leaf], dy.float())
    assert torch.equal(y, cp4.mx4_linear(x.float(), q, dense.bias)) and torch.equal(dx, cp4.mx4_linear_backward(dy.float(), q))
    traced = torch.jit.trace(dense, (x.float(),), check_trace=False)
    z = torch.randn(300, 70, device="cuda")
    assert torch.equal(traced(z), dense(z))
    assert dense.bfloat16().bias.dtype == torch.float32
    fast = torch_ops.Mx4Linear(W, bias, activations=4)
    assert torch.equal(fast(z), cp4.mx4_linear(z, q, fast.bias, activations=4))
    with pytest.raises(ValueError, match="no gradient"):
        fast(leaf)
    with pytest.raises(ValueError, match="not trained"):
        torch_ops.mx4_linear(leaf, q, torch.zeros(48, device="cuda", requires_grad=True))


def test_streams_and_graph(cp4):
    q, _ = weights(cp4, 300, 520, torch.bfloat16)
    x, dy = make(200, 520, dtype=torch.bfloat16), make(200, 300, dtype=torch.bfloat16, seed=2)
    run = lambda **kw: (cp4.mx4_linear(x, q, **kw), cp4.mx4_linear(x, q, activations=4, **kw), cp4.mx4_linear_backward(dy, q, **kw),  # noqa: E731
                        cp4.mx4_linear(x[:5], q, **kw), cp4.mx4_dequantize(cp4.mx4_quantize(x, **kw), **kw))
    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = run(stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for seed in range(3):
        x.copy_(make(200, 520, dtype=torch.bfloat16, seed=seed))
        dy.copy_(make(200, 300, dtype=torch.bfloat16, seed=seed + 9))
        graph.replay()
        want = run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals(cp4):
    q, _ = weights(cp4, 40, 64, torch.float32)
    x = make(4, 64)
    both = torch.zeros(256, dtype=torch.uint8, device="cuda")
    bad = [lambda: cp4.mx4_quantize(x.cpu()), lambda: cp4.mx4_quantize(x.double()), lambda: cp4.mx4_quantize(x[:, :0]),
           lambda: cp4.mx4_linear(x[:, :63], q), lambda: cp4.mx4_linear(x.double(), q), lambda: cp4.mx4_linear(x, q, torch.zeros(39, device="cuda")),
           lambda: cp4.mx4_linear(x, cp4.Mx4(q.codes, q.scales, 97)), lambda: cp4.mx4_linear(x, cp4.Mx4(q.codes[:, :31], q.scales, 64)),
           lambda: cp4.mx4_linear(x, cp4.Mx4(q.codes, q.scales[:39], 64)), lambda: cp4.mx4_linear(x, cp4.Mx4(q.codes.cpu(), q.scales.cpu(), 64)),
           lambda: cp4.mx4_linear(x, cp4.Mx4(q.codes.int(), q.scales, 64)), lambda: cp4.mx4_linear(x, q.codes), lambda: cp4.mx4_linear(x, q, dtype=torch.float16),
           lambda: cp4.mx4_linear(x, q, out=torch.zeros(4, 39, device="cuda")), lambda: cp4.mx4_linear_backward(x, q),
           lambda: cp4.mx4_dequantize(q, torch.float64), lambda: cp4.mx4_dequantize(q, torch.float32, torch.zeros(40, 63, device="cuda")),
           lambda: cp4.mx4_linear(cp4.mx4_quantize(make(4, 63)), q), lambda: cp4.mx4_linear(x, q, out=x.view(-1)[:160].view(4, 40)),
           lambda: cp4.mx4_dequantize(cp4.Mx4(both[:32].view(2, 16), both[32:34].view(2, 1), 16), out=both.view(torch.float32)[:32].view(2, 16))]
    for call in bad:
        with pytest.raises(AssertionError):
            call()
    for call in (lambda: cp4.mx4_linear(x, q, activations=8), lambda: __import__("paralleltnnlayers_amd.torch_ops").torch_ops.AdapterLinear(64, 40, 4, weight_bits=8)):
        with pytest.raises(ValueError):
            call()


def test_rows_of_another_length_are_refused_in_a_trace(cp4):
    from paralleltnnlayers_amd import torch_ops
    q, _ = weights(cp4, 40, 60, torch.float32)
    A, B, ids = make(1, 4, 64), make(1, 40, 4), torch.zeros(4, dtype=torch.int32, device="cuda")
    for call in (lambda x: torch_ops.mx4_linear(x, q), lambda x: torch_ops.adapter_linear(x, q, A, B, ids)):
        with pytest.raises(AssertionError):
            call(make(4, 64))
        with pytest.raises(AssertionError):
            torch.jit.trace(call, (make(4, 64),), check_trace=False)
