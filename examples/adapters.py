"""Low-rank adapters on a frozen classifier behind a CP convolution: trained, then served.

A small image network - a CP4 convolution, its mean over the plane, a frozen dense classifier - is given to
several users, each with labels of their own.  One low-rank adapter a user is trained on a batch that
holds everybody's images (``torch_ops.AdapterLinear`` and ``optim.AdamW``, moments in 8 bits, gradients
clipped by their norm), and the trained adapters then answer a batch of mixed requests in one call.  With ``--four``
the features pass a layer norm, the classifier is held in 4 bits, and the adapters are trained by ``optim.Muon``.

    python examples/adapters.py [--users 8] [--steps 60] [--four]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import paralleltnnlayers_amd as cp4  # noqa: E402
from paralleltnnlayers_amd import optim, torch_ops  # noqa: E402


class Network(torch.nn.Module):
    def __init__(self, users, features=64, classes=10, rank=8, four=False):
        super().__init__()
        self.conv = torch_ops.CP4Conv2d(3, features, 3, 16, bias=True, activation="relu")
        self.head = torch_ops.AdapterLinear(features, classes, rank=rank, adapters=users, weight_bits=4 if four else None)
        self.norm = torch_ops.LayerNorm(features) if four else torch.nn.Identity()

    def features(self, images):
        return self.norm(self.conv(images).mean(dim=(2, 3)))

    def forward(self, images, user):
        return self.head(self.features(images), user)


def run(users=8, steps=60, images=256, size=24, seed=0, four=False):
    """(loss before, loss after, share of a mixed batch's answers that serving and training agree on)."""
    torch.manual_seed(seed)
    net = Network(users, four=four)
    x = torch.randn(images, 3, size, size, device="cuda")
    user = torch.randint(0, users, (images,), device="cuda", dtype=torch.int32)
    label = (x.mean(dim=(1, 2, 3)).argsort().argsort() * 10 // images + user) % 10   # each user counts from another class
    adapters = [net.head.A, net.head.B] if four else []
    rest = [p for p in net.parameters() if all(p is not a for a in adapters)]
    opts = [optim.AdamW(rest, lr=2e-2, weight_decay=0.0, state_bits=8, min_8bit_size=256, max_norm=1.0)]
    if four:
        opts.append(optim.Muon(adapters, lr=2e-2))
    losses = []
    for _ in range(steps):
        net.zero_grad()
        loss = torch.nn.functional.cross_entropy(net(x, user), label)
        loss.backward()
        for opt in opts:
            opt.step()
        losses.append(float(loss.detach()))
    torch_ops.check_device()

    # serving: the adapters of all users beside the one classifier, requests in any order, some without an adapter
    with torch.no_grad():
        h = net.head
        mixed = torch.where(torch.arange(images, device="cuda") % 5 == 0, torch.full_like(user, -1), user)
        feats = net.features(x)
        served = cp4.adapter_forward(feats, h.projection(), h.A, h.B, mixed, scale=h.scale)
        weight = cp4.mx4_dequantize(h.projection()) if four else h.weight
        alone = torch.where((mixed >= 0)[:, None], net(x, user), feats @ weight.t())
    agree = float((served.argmax(1) == alone.argmax(1)).float().mean())
    return losses[0], losses[-1], agree


if __name__ == "__main__":
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--users", type=int, default=8)
    p.add_argument("--steps", type=int, default=60)
    p.add_argument("--four", action="store_true")
    a = p.parse_args()
    before, after, agree = run(a.users, a.steps, four=a.four)
    print(f"loss {before:.3f} -> {after:.3f}; served answers as trained: {100 * agree:.1f} %")
