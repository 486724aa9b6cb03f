"""What the speed of the low-rank adapters and of the AdamW step is measured on.

Three operators:

* ``serve``: a shared projection with the low-rank adapters of many requests beside it,
  ``y[t] = W x[t] + bias + s_a B_a (A_a x[t])`` with ``a = ids[t]``; an id of -1 is a token
  without an adapter;
* ``train``: the same layer trained: its output, then the gradients of the input and of all
  adapters (``W`` and the bias are frozen);
* ``adamw``: one AdamW step over many tensors, its moments held in 32 bits or in 8.

8-bit moments: each 256 consecutive values of a tensor share the float32 scale ``s``, their
largest magnitude.  The first moment is an int8 ``q`` that stands for ``sign(q) q^2 s / 127^2``,
the second a uint8 that stands for ``q^4 s / 255^4``; both are rounded to nearest in ``q``, and a
second moment above zero has a ``q`` of at least 1.

Sizes are generic, or those of the dense layers behind the convolutions of AlexNet and VGG-16
(9216 and 25088 inputs, 4096 units, 1000 classes) and of the factors of VGG-16's convolutions.
``draw`` covers what lies between: 1 to 8192 tokens, 64 to 25088 inputs and 64 to 8192 outputs,
odd ones among them, ranks 1 to 64, 1 to 64 adapters, fp32 and both 16-bit types; 1 to 200
tensors of 1000 to 128 million values together.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BLOCK = 256        # values that share a scale
LIMIT = 8192 * 4096 * 4096   # tokens * inputs * outputs of the largest layer


def _layer(name, op, T, K, N, R, G, requests, dtype, bias=False):
    return dict(name=name, op=op, T=T, K=K, N=N, R=R, G=G, requests=requests, dtype=dtype, bias=bias)


def _adamw(name, kind, layers, K, N, R, param, grad, bits, clip=False, copy=""):
    return dict(name=name, op="adamw", kind=kind, layers=layers, K=K, N=N, R=R, param=param, grad=grad,
                bits=bits, clip=clip, copy=copy)


def listed():
    return [
        # one new token of one request: nothing but latency
        _layer("serve_1x1024x1024_r8_bf16", "serve", 1, 1024, 1024, 8, 4, 1, "bf16"),
        # a step of 48 requests, one new token each, most with an adapter of their own
        _layer("serve_48x4096x4096_r16_bf16", "serve", 48, 4096, 4096, 16, 32, 48, "bf16"),
        # prompts of many lengths and single tokens in one batch, an odd number of tokens
        _layer("serve_2077x4096x8192_r32_bf16", "serve", 2077, 4096, 8192, 32, 16, 40, "bf16", bias=True),
        # AlexNet's first dense layer on a few images, the framework's own type
        _layer("serve_16x9216x4096_r16_f32", "serve", 16, 9216, 4096, 16, 8, 16, "f32", bias=True),
        # a classifier with nothing even about it: rows that start anywhere
        _layer("serve_333x1001x777_r5_f16", "serve", 333, 1001, 777, 5, 7, 60, "f16", bias=True),
        # VGG-16's first dense layer, one adapter trained on a batch of 64 images
        _layer("train_64x25088x4096_r16_f32", "train", 64, 25088, 4096, 16, 1, 1, "f32"),
        # rank 64 in half precision, an odd number of tokens, adapters trained side by side
        _layer("train_1031x2048x2816_r64_f16", "train", 1031, 2048, 2816, 64, 4, 9, "f16", bias=True),
        # the largest batch: eight adapters trained on one projection
        _layer("train_8192x4096x4096_r16_bf16", "train", 8192, 4096, 4096, 16, 8, 16, "bf16"),
        # the CP factors and biases of VGG-16's convolutions: tens of tiny tensors
        _adamw("adamw_factors_r16_32", "factors", 13, 0, 0, 16, "f32", "f32", 32),
        # dense layers in 16 bits over float32 masters, gradients clipped by their norm
        _adamw("adamw_dense_50M_32_clip", "dense", 12, 2048, 2048, 0, "f32", "bf16", 32, clip=True, copy="bf16"),
        # adapters of many projections, moments in 8 bits, odd sizes
        _adamw("adamw_adapters_r7_8", "adapters", 28, 1001, 777, 7, "f32", "f32", 8),
        # the largest: 134 million values, moments in 8 bits
        _adamw("adamw_dense_134M_8", "dense", 8, 4096, 4096, 0, "f32", "bf16", 8),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("serve", "train", "adamw"))
    if op == "adamw":
        bits = rng.choice((32, 8))
        param, grad, copy = rng.choice((("f32", "f32", ""), ("f32", "bf16", "bf16"), ("bf16", "bf16", ""),
                                        ("f32", "f16", "f16")))
        kind = rng.choice(("factors", "adapters", "dense"))
        while True:
            c = _adamw("", kind, _log(rng, 1, 40), _log(rng, 32, 4096), _log(rng, 32, 4096), rng.randint(1, 64),
                       param, grad, bits, bits == 32 and rng.random() < 0.5, copy)
            if 1000 <= sum(_sizes(c)) <= 8 * (4096 * 4096 + 4096) and 3072 not in (c["K"], c["N"]):
                break
    else:
        while True:
            T, K, N = _log(rng, 1, 8192), _log(rng, 64, 25088), _log(rng, 64, 8192)
            if rng.random() < 0.6:      # most layers have even sizes
                K, N = max(64, K // 64 * 64), max(64, N // 64 * 64)
            if T * K * N <= LIMIT and 3072 not in (T, K, N):
                break
        c = _layer("", op, T, K, N, rng.choice((rng.randint(1, 64), 8, 16, 32)), _log(rng, 1, 64),
                   min(T, _log(rng, 1, 64)), rng.choice(("f32", "bf16", "f16")), rng.random() < 0.5)
    del c["name"]
    return c


# ---- sizes and work ------------------------------------------------------------------

# out and in channels of VGG-16's convolutions
_CONVS = ((64, 3), (64, 64), (128, 64), (128, 128), (256, 128), (256, 256), (256, 256), (512, 256), (512, 512),
          (512, 512), (512, 512), (512, 512), (512, 512))


def _sizes(c):
    """The number of values of each tensor of an AdamW step."""
    if c["kind"] == "factors":       # FK, FC, FH, FW and the bias of each convolution
        every = [_CONVS[i % len(_CONVS)] for i in range(c["layers"])]
        return [n for t, k in every for n in (t * c["R"], k * c["R"], 3 * c["R"], 3 * c["R"], t)]
    if c["kind"] == "adapters":
        return [c["R"] * c["K"], c["N"] * c["R"]] * c["layers"]
    return [c["K"] * c["N"], c["N"]] * c["layers"]


def _starts(sizes):
    """Where each tensor starts in the flat buffer: at whole blocks."""
    ends = np.cumsum([-(-n // BLOCK) * BLOCK for n in sizes])
    return [0] + [int(e) for e in ends[:-1]], int(ends[-1])


def work(c):
    if c["op"] == "adamw":
        n = sum(_sizes(c))
        state = 16 if c["bits"] == 32 else 4 + 8 + 16 / BLOCK     # 8 bits: and their values, written
        copy = DTYPES[c["copy"]].itemsize if c["copy"] else 0
        return {"bytes": n * (2 * DTYPES[c["param"]].itemsize + DTYPES[c["grad"]].itemsize + state + copy),
                "flops": 15 * n}
    T, K, N, R, e = c["T"], c["K"], c["N"], c["R"], DTYPES[c["dtype"]].itemsize
    if c["op"] == "serve":
        used = min(c["G"], c["requests"])
        return {"bytes": e * (T * K + N * K + T * N + used * R * (K + N)) + 4 * T,
                "flops": 2 * T * N * K + 2 * T * R * (K + N)}
    return {"bytes": e * (2 * T * K + N * K + 2 * T * N + 2 * c["G"] * R * (K + N)) + 4 * T,
            "flops": 4 * T * N * K + 6 * T * R * (K + N)}


# ---- inputs -----------------------------------------------------------------------------

def _ids(c, seed):
    """The adapter of each token: requests one after the other, one in eight without an adapter."""
    r = np.random.RandomState(seed % (1 << 31))
    T, q = c["T"], c["requests"]
    cuts = np.sort(r.choice(np.arange(1, T), q - 1, replace=False)) if q > 1 else np.zeros(0, np.int64)
    lengths = np.diff(np.concatenate([[0], cuts, [T]]))
    of = np.where(r.rand(q) < (0.125 if q > 1 else 0.0), -1, r.randint(0, c["G"], q))
    return torch.from_numpy(np.repeat(of, lengths).astype(np.int32)).cuda()


def prepare(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)

    if c["op"] != "adamw":
        T, K, N, R, G, dtype = c["T"], c["K"], c["N"], c["R"], c["G"], DTYPES[c["dtype"]]
        s = {"case": c, "x": normal(T, K, dtype=dtype), "W": normal(N, K, std=K ** -0.5, dtype=dtype),
             "A": normal(G, R, K, std=K ** -0.5, dtype=dtype), "B": normal(G, N, R, std=R ** -0.5, dtype=dtype),
             "scale": 0.25 + torch.rand(G, device="cuda", generator=g), "ids": _ids(c, int(seed)),
             "bias": normal(N) if c["bias"] else None}
        if c["op"] == "train":
            s["dy"] = normal(T, N, dtype=dtype)
            for k in ("x", "A", "B"):
                s[k].requires_grad_(True)
        return s

    sizes = _sizes(c)
    starts, total = _starts(sizes)
    real = torch.zeros(total, dtype=torch.bool)
    for at, n in zip(starts, sizes):
        real[at:at + n] = True
    real = real.cuda()
    steps, beta1, beta2 = 100 + int(seed) % 1000, 0.9, 0.999

    # gradients spread over several powers of ten; each moment goes with its own value's
    size = normal(total, std=1.5).exp_().mul_(1e-3)
    p = normal(total, std=0.05).mul_(real).to(DTYPES[c["param"]])
    m = normal(total, std=0.3).mul_(size).mul_(real)
    v = size.square().mul_(0.5 + torch.rand(total, device="cuda", generator=g)).mul_(real)
    s = {"case": c, "p": p, "g": normal(total).mul_(size).mul_(real).to(DTYPES[c["grad"]]),
         "counter": torch.tensor([steps, beta1 ** steps, beta2 ** steps, 0.0], dtype=torch.float64, device="cuda"),
         "hyper": dict(lr=1e-3, betas=(beta1, beta2), eps=1e-8, weight_decay=0.01)}
    if c["bits"] == 32:
        s["m"], s["v"] = m, v
    else:
        s["m"], s["v"], s["scales"] = _codes(m, v)
        s["m_values"], s["v_values"] = torch.zeros(total, device="cuda"), torch.zeros(total, device="cuda")
    if c["copy"]:
        s["copy"] = p.to(DTYPES[c["copy"]])
    if c["clip"]:
        s["hyper"]["max_norm"] = 1.0
    # the tensors that the program has: pieces of the buffers
    cut = lambda t: [t[at:at + n] for at, n in zip(starts, sizes)]  # noqa: E731
    s["lists"] = {k: cut(s[k]) for k in ("p", "g", "m", "v", "copy", "m_values", "v_values") if k in s}
    if c["bits"] == 8:
        s["lists"]["scales"] = [s["scales"][:, at // BLOCK:at // BLOCK - (-n // BLOCK)] for at, n in zip(starts, sizes)]
    return s


# ---- one pass --------------------------------------------------------------------------------

def run(s):
    return {"serve": _serve, "train": _train, "adamw": _step}[s["case"]["op"]](s)


def _serve(s):
    if own:
        import paralleltnnlayers_amd as cp4

        return cp4.adapter_forward(s["x"], s["W"], s["A"], s["B"], s["ids"], scale=s["scale"], bias=s["bias"])
    return _plain_forward(s)[0].to(s["x"].dtype)


def _train(s):
    if own:
        from paralleltnnlayers_amd import torch_ops

        y = torch_ops.adapter_linear(s["x"], s["W"], s["A"], s["B"], s["ids"], scale=s["scale"], bias=s["bias"])
        return (y.detach(),) + torch.autograd.grad(y, (s["x"], s["A"], s["B"]), s["dy"])
    with torch.no_grad():
        y, h, mask, (x, W, A, B) = _plain_forward(s)
        (G, R, K), N, dy = s["A"].shape, s["W"].shape[0], s["dy"].float()
        dh = dy @ B * mask                                        # [T, G * R]
        dx = dy @ W + dh @ A
        dA, dB = dh.t() @ x, (dy.t() @ h).view(N, G, R).permute(1, 0, 2)
        t = s["x"].dtype
        return y.to(t), dx.to(t), dA.view(G, R, K).to(t), dB.to(t).contiguous()


def _plain_forward(s):
    """y in 32 bits, and what the gradients need: every token against every adapter, masked."""
    with torch.no_grad():
        (G, R, K), N = s["A"].shape, s["W"].shape[0]
        x, W, A = s["x"].float(), s["W"].float(), s["A"].float().view(G * R, K)
        B = s["B"].float().permute(1, 0, 2).reshape(N, G * R)
        mask = (s["ids"][:, None] == torch.arange(G, device="cuda")) * s["scale"]
        mask = mask.repeat_interleave(R, dim=1)                   # [T, G * R]: the scale of the token's own adapter
        h = x @ A.t() * mask
        y = x @ W.t() + h @ B.t()
        if s["bias"] is not None:
            y = y + s["bias"]
        return y, h, mask, (x, W, A, B)


def _step(s):
    if own:
        from paralleltnnlayers_amd import optim

        of = s["lists"]
        norm = optim.adamw_step(of["p"], of["g"], of["m"], of["v"], s["counter"], scales=of.get("scales"),
                                copies=of.get("copy"), **s["hyper"])
        if s["case"]["bits"] == 8:
            optim.moment_values(of["m"], of["v"], of["scales"], out=(of["m_values"], of["v_values"]))
    else:
        norm = _plain_step(s)
    m, v = ("m_values", "v_values") if s["case"]["bits"] == 8 else ("m", "v")
    return {"p": s["p"], "m": s[m], "v": s[v], "counter": s["counter"][:3], "copy": s.get("copy"), "norm": norm}


def _plain_step(s):
    h, c, eight = s["hyper"], s["counter"], s["case"]["bits"] == 8
    beta1, beta2 = h["betas"]
    g, norm = s["g"].float(), None
    if "max_norm" in h:
        norm = (g * g).sum().sqrt()
        g = g * (h["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    power1, power2 = c[1] * beta1, c[2] * beta2                   # beta ** steps, in 64 bits
    rate, root = (h["lr"] / (1 - power1)).float(), (1 / (1 - power2).sqrt()).float()
    m, v = (_values(s) if eight else (s["m"], s["v"]))
    m = m * beta1 + g * (1 - beta1)
    v = v * beta2 + (g * g) * (1 - beta2)
    p = s["p"].float() * (1 - h["lr"] * h["weight_decay"]) - (m / (v.sqrt() * root + h["eps"])) * rate
    s["p"].copy_(p)
    if "copy" in s:
        s["copy"].copy_(p)
    c[:3] = torch.stack([c[0] + 1, power1, power2])
    if eight:
        for k, t in zip(("m", "v", "scales"), _codes(m, v)):
            s[k].copy_(t)
        m, v = _values(s)
        s["m_values"].copy_(m)
        s["v_values"].copy_(v)
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
    return norm


def _codes(m, v):
    """The 8-bit codes of two moments and their scales; a scale below the smallest normal number is none."""
    m, v = m.view(-1, BLOCK), v.view(-1, BLOCK)
    tops = torch.stack([m.abs().amax(1), v.amax(1)])
    tops = torch.where(tops >= 2.0 ** -126, tops, torch.zeros_like(tops))
    over = torch.where(tops > 0, 1 / tops, tops)[:, :, None]
    qm = ((m.abs() * over[0]).sqrt() * 127).round() * m.sign()
    qv = ((v * over[1]).sqrt().sqrt() * 255).round()
    qv = torch.where((qv < 1) & (v > 0) & (over[1] > 0), torch.ones_like(qv), qv)
    return qm.to(torch.int8).view(-1), qv.to(torch.uint8).view(-1), tops


def _values(s):
    """What the 8-bit moments stand for."""
    m, v = s["m"].float().view(-1, BLOCK), s["v"].float().view(-1, BLOCK)
    tops = s["scales"][:, :, None]
    m = m.abs() * m * (tops[0] * (1 / 127 ** 2))
    v2 = v * v
    return m.reshape(-1), (v2 * v2 * (tops[1] * (1 / 255 ** 4))).reshape(-1)


# ---- the definition, in 64 bits -----------------------------------------------------------

def exact(c, seed):
    s = prepare(c, seed)
    with torch.no_grad():
        return _exact_step(s) if c["op"] == "adamw" else _exact_layer(s)


def _exact_layer(s):
    x, W, scale = s["x"].double(), s["W"].double(), s["scale"].double()
    y = torch.nn.functional.linear(x, W)
    if s["bias"] is not None:
        y += s["bias"].double()
    train = s["case"]["op"] == "train"
    if train:
        dy = s["dy"].double()
        dx = torch.mm(dy, W)
        dA, dB = torch.zeros(s["A"].shape, dtype=torch.float64, device="cuda"), torch.zeros(s["B"].shape, dtype=torch.float64, device="cuda")
    for a in range(s["A"].shape[0]):                      # the tokens of one adapter at a time
        at = (s["ids"] == a).nonzero().flatten()
        A, B = s["A"][a].double(), s["B"][a].double()
        xa = x.index_select(0, at)
        y.index_add_(0, at, torch.mm(torch.mm(xa, A.t()), B.t()) * scale[a])
        if train:
            dya = dy.index_select(0, at)
            dx.index_add_(0, at, torch.mm(torch.mm(dya, B), A) * scale[a])
            dB[a] = torch.mm(dya.t(), torch.mm(xa, A.t())) * scale[a]
            dA[a] = torch.mm(torch.mm(dya, B).t(), xa) * scale[a]
    return (y, dx, dA, dB) if train else y


def _exact_step(s):
    h, c, eight = s["hyper"], s["counter"].tolist(), s["case"]["bits"] == 8
    beta1, beta2 = h["betas"]
    t = int(c[0]) + 1
    g, p, norm = s["g"].double(), s["p"].double(), None
    if "max_norm" in h:
        norm = torch.linalg.vector_norm(g)
        g = g * min(1.0, h["max_norm"] / (float(norm) + 1e-6))
    m, v = s["m"].double(), s["v"].double()
    if eight:
        tops = s["scales"].double().repeat_interleave(BLOCK, dim=1)
        m, v = m * m.abs() / 127.0 ** 2 * tops[0], (v / 255.0) ** 4 * tops[1]
    m, v = torch.lerp(g, m, beta1), torch.lerp(g.square(), v, beta2)
    step = h["lr"] * (m / (1 - beta1 ** t)) / ((v / (1 - beta2 ** t)).sqrt() + h["eps"])
    p = p - h["lr"] * h["weight_decay"] * p - step
    if eight:
        m, v = _nearest(m, 127, 2, 0), _nearest(v, 255, 4, 1)
    counter = torch.tensor([t, beta1 ** t, beta2 ** t], dtype=torch.float64)
    return {"p": p, "m": m, "v": v, "counter": counter, "copy": p if "copy" in s else None, "norm": norm}


def _nearest(x, levels, power, least):
    """Each value's nearest level (nearest before it is raised to ``power``) of its block."""
    x = x.view(-1, BLOCK)
    top = x.abs().amax(dim=1, keepdim=True)
    edges = ((torch.arange(levels, dtype=torch.float64, device="cuda") + 0.5) / levels) ** power
    q = torch.searchsorted(edges, (x.abs() / top.clamp(min=1e-300)).contiguous()).double()
    q = torch.where((x != 0) & (q < least), torch.full_like(q, least), q)
    return ((q / levels) ** power * top * x.sign()).reshape(-1)
