"""Low-rank adapters on a frozen classifier behind a CP convolution: trained, then served.

A small image network - a CP4 convolution, its mean over the plane, a frozen dense classifier - is given to
several users, each with labels of their own.  One low-rank adapter a user is trained on a batch that
holds everybody's images (``torch_ops.AdapterLinear`` and ``optim.AdamW``, moments in 8 bits, gradients
clipped by their norm), and the trained adapters then answer a batch of mixed requests in one call.

    python examples/adapters.py [--users 8] [--steps 60]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import paralleltnnlayers_amd as cp4  # noqa: E402
from paralleltnnlayers_amd import optim, torch_ops  # noqa: E402


class Network(torch.nn.Module):
    def __init__(self, users, features=64, classes=10, rank=8):
        super().__init__()
        self.conv = torch_ops.CP4Conv2d(3, features, 3, 16, bias=True, activation="relu")
        self.head = torch_ops.AdapterLinear(features, classes, rank=rank, adapters=users)

    def features(self, images):
        return self.conv(images).mean(dim=(2, 3))

    def forward(self, images, user):
        return self.head(self.features(images), user)


def run(users=8, steps=60, images=256, size=24, seed=0):
    """(loss before, loss after, share of a mixed batch's answers that serving and training agree on)."""
    torch.manual_seed(seed)
    net = Network(users)
    x = torch.randn(images, 3, size, size, device="cuda")
    user = torch.randint(0, users, (images,), device="cuda", dtype=torch.int32)
    label = (x.mean(dim=(1, 2, 3)).argsort().argsort() * 10 // images + user) % 10   # each user counts from another class
    opt = optim.AdamW(net.parameters(), lr=2e-2, weight_decay=0.0, state_bits=8, min_8bit_size=256, max_norm=1.0)
    losses = []
    for _ in range(steps):
        opt.zero_grad()
        loss = torch.nn.functional.cross_entropy(net(x, user), label)
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
    torch_ops.check_device()

    # serving: the adapters of all users beside the one classifier, requests in any order, some without an adapter
    with torch.no_grad():
        h = net.head
        mixed = torch.where(torch.arange(images, device="cuda") % 5 == 0, torch.full_like(user, -1), user)
        feats = net.features(x)
        served = cp4.adapter_forward(feats, h.weight, h.A, h.B, mixed, scale=h.scale)
        alone = torch.where((mixed >= 0)[:, None], net(x, user), feats @ h.weight.t())
    agree = float((served.argmax(1) == alone.argmax(1)).float().mean())
    return losses[0], losses[-1], agree


if __name__ == "__main__":
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--users", type=int, default=8)
    p.add_argument("--steps", type=int, default=60)
    a = p.parse_args()
    before, after, agree = run(a.users, a.steps)
    print(f"loss {before:.3f} -> {after:.3f}; served answers as trained: {100 * agree:.1f} %")
