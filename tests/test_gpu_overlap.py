"""An output that the caller gives is none of the operands' memory (but x itself, of a layer norm); what only looks like it runs."""
import pytest
import torch

pytestmark = pytest.mark.gpu
T, K, N = 6, 64, 64


@pytest.fixture(scope="module")
def cp4():
    import paralleltnnlayers_amd as cp4
    cp4.lib()
    return cp4


def part(room, first, *shape, dtype=torch.float32):
    """A contiguous tensor in a uint8 room, from byte ``first`` on."""
    size = torch.empty(0, dtype=dtype).element_size()
    for n in shape:
        size *= n
    return room[first:first + size].view(dtype).view(shape)


def refused(room, call):
    before = room.clone()
    with pytest.raises(AssertionError, match="overlaps"):
        call()
    assert torch.equal(room, before)


def test_layer_norm(cp4):
    room = torch.randint(0, 60, (1 << 14,), dtype=torch.uint8, device="cuda")
    D = 32
    x = part(room, 0, T, D)
    wide = part(room, 0, T, 2 * D)[:, :D]
    w, b = part(room, 8192, D), part(room, 8192 + 4 * D, D)
    # behind x by a row, within a strided x, over weight and bias, over x's last value
    for call in (lambda: cp4.layer_norm_forward(x, w, b, out=part(room, 4 * D, T, D)),
                 lambda: cp4.layer_norm_forward(wide, w, b, out=part(room, 0, T, D)),
                 lambda: cp4.layer_norm_forward(wide, w, b, out=part(room, 4 * D, T, D)),
                 lambda: cp4.layer_norm_forward(x, w, b, out=part(room, 8192 - 4 * D, T, D)),
                 lambda: cp4.layer_norm_forward(x, None, b, out=part(room, 8192 + 4 * D, T, D)),
                 lambda: cp4.layer_norm_forward(x, w, b, out=part(room, 4 * T * D - 4, T, D))):
        refused(room, call)
    want = cp4.layer_norm_forward(x, w, b)
    near = part(room, 4 * T * D, T, D)                               # right behind it
    assert torch.equal(cp4.layer_norm_forward(x, w, b, out=near), want)
    assert torch.equal(cp4.layer_norm_forward(x.view(2, 3, D), w, b, out=x).view(T, D), want) and torch.equal(x, want)
    assert cp4.layer_norm_forward(x[:0], w, b, out=part(room, 8192, 0, D)).shape == (0, D)


def test_projections_in_4_bits(cp4):
    torch.manual_seed(0)
    q = cp4.mx4_quantize(torch.randn(N, K, device="cuda"))
    room = torch.zeros(1 << 15, dtype=torch.uint8, device="cuda")
    codes, scales, bias = part(room, 0, N, K // 2, dtype=torch.uint8), part(room, 2048, N, K // 32, dtype=torch.uint8), part(room, 4096, N)
    codes.copy_(q.codes)
    scales.copy_(q.scales)
    bias.normal_()
    x = part(room, 8192, T, K)
    x.normal_()
    W, xq = cp4.Mx4(codes, scales, K), cp4.mx4_quantize(x)
    px = cp4.Mx4(part(room, 16384, T, K // 2, dtype=torch.uint8), part(room, 17408, T, K // 32, dtype=torch.uint8), K)
    px.codes.copy_(xq.codes)
    px.scales.copy_(xq.scales)
    for at in (0, 1024, 2048 - 256, 2048, 4096, 4096 - 1024):        # codes, scales, bias
        out = part(room, at, T, N)
        for args in ((x, W, bias), (px, W, bias)):
            refused(room, lambda: cp4.mx4_linear(*args, out=out))
        refused(room, lambda: cp4.mx4_linear(x, W, bias, activations=4, out=out))
    refused(room, lambda: cp4.mx4_linear(x, W, bias, out=part(room, 8192 + 256, T, N)))
    refused(room, lambda: cp4.mx4_linear(px, W, out=part(room, 16384, T, N)))
    refused(room, lambda: cp4.mx4_linear(px, W, out=part(room, 17408 - 512, T, N)))
    refused(room, lambda: cp4.mx4_dequantize(W, out=part(room, 2048, N, K)))
    free = part(room, 20480, T, N)
    assert torch.equal(cp4.mx4_linear(x, W, bias, out=free), cp4.mx4_linear(x, q, bias))
    assert torch.equal(cp4.mx4_linear(px, W, bias, out=free), cp4.mx4_linear(xq, q, bias))
    # (x rounded to 4 bits is read before y is written)
    want = cp4.mx4_linear(x, q, bias, activations=4)
    assert torch.equal(cp4.mx4_linear(x, W, bias, activations=4, out=x), want)


@pytest.mark.parametrize("four", [False, True])
def test_projections_with_adapters(cp4, four):
    torch.manual_seed(0)
    R, G = 4, 2
    room = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    sizes = dict(x=(T, K), W=(N, K), A=(G, R, K), B=(G, N, R), scale=(G,), bias=(N,), out=(T, N))
    at, t = 0, {}
    for k, s in sizes.items():
        t[k] = part(room, at, *s)
        t[k].normal_()
        at += (t[k].numel() * 4 + 4096 + 255) // 256 * 256
    ids = part(room, at, T, dtype=torch.int32)
    ids.copy_(torch.tensor([0, 1, -1, 1, 0, 0]))
    W = t["W"]
    if four:
        q = cp4.mx4_quantize(W)
        W = cp4.Mx4(part(room, at + 4096, *q.codes.shape, dtype=torch.uint8), part(room, at + 8192, *q.scales.shape, dtype=torch.uint8), K)
        W.codes.copy_(q.codes)
        W.scales.copy_(q.scales)
    run = lambda out: cp4.adapter_forward(t["x"], W, t["A"], t["B"], ids, t["scale"], t["bias"], out=out)  # noqa: E731
    starts = [t[k].data_ptr() - room.data_ptr() for k in ("x", "A", "B", "scale", "bias")] + [ids.data_ptr() - room.data_ptr()]
    starts += [w.data_ptr() - room.data_ptr() for w in (W[:2] if four else [W])]
    for first in starts:
        for shift in (0, -1024):
            if first + shift >= 0:
                refused(room, lambda: run(part(room, first + shift, T, N)))
    want = cp4.adapter_forward(t["x"].clone(), W, t["A"].clone(), t["B"], ids, t["scale"], t["bias"])
    assert torch.equal(run(t["out"]), want)
