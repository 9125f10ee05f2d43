"""A network over the points of packed molecules, trained to tell the elements of atoms that were masked from what is around them:

    elements  ->  embedding  ->  blocks: u + attention(linear(norm(u))) by distance, u + linear(act(linear(norm(u))))
              ->  linear_cross_entropy of the masked atoms

Molecules lie one behind the other (starts); atoms see those of their own molecule.  Only distances between points enter, so that nothing changes
when a molecule is turned or moved.  All weights are changed by one AdamW step.

    python examples/elements.py [--steps 40] [--bfloat16]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import gelib_amd as gelib  # noqa: E402


class Elements(torch.nn.Module):

    def __init__(self, elements=16, width=64, heads=8, kv_heads=4, blocks=2, dtype=torch.float32, device="cuda"):
        super().__init__()
        self.heads, self.kv, self.dim = heads, kv_heads, width // heads

        def real(*shape, scale=0.0, at=0.0):
            return torch.nn.Parameter((at + scale * torch.randn(*shape, device=device)).to(dtype))
        self.table = real(elements + 1, width, scale=1.0)   # the last row: masked
        columns = (heads + 2 * kv_heads) * self.dim
        self.blocks = torch.nn.ModuleList()
        for _ in range(blocks):
            b = torch.nn.Module()
            b.gain, b.shift, b.qkv, b.out = real(width, at=1.0), real(width), real(width, columns, scale=width ** -0.5), real(width, width, scale=width ** -0.5)
            b.slopes = torch.nn.Parameter(torch.linspace(0.2, 2.0, heads, device=device))
            b.gain2, b.shift2, b.up, b.down = real(width, at=1.0), real(width), real(width, 2 * width, scale=width ** -0.5), real(2 * width, width, scale=(2 * width) ** -0.5)
            self.blocks.append(b)
        self.last, self.bias = real(width, elements, scale=width ** -0.5), real(elements)

    def features(self, tokens, points, starts):
        u = gelib.embedding(tokens, self.table)
        for b in self.blocks:
            qkv = gelib.linear_act(gelib.group_norm_act(u, 1, b.gain, b.shift), b.qkv).view(len(u), -1, self.dim)
            q, k, v = qkv[:, :self.heads], qkv[:, self.heads:self.heads + self.kv], qkv[:, self.heads + self.kv:]
            u = gelib.linear_act(gelib.attention(q, k, v, points, b.slopes, starts=starts).reshape(u.shape), b.out, residual=u)
            u = gelib.linear_act(gelib.linear_act(gelib.group_norm_act(u, 1, b.gain2, b.shift2), b.up, act="gelu"), b.down, residual=u)
        return u

    def forward(self, tokens, points, starts, targets):
        """Losses of the atoms with a target; zero of the others (targets below zero)."""
        return gelib.linear_cross_entropy(self.features(tokens, points, starts), self.last, targets, self.bias)


def data(molecules, elements, seed, device="cuda"):
    """Random molecules: how many atoms each has, their places and elements, every sixth or so masked.  An atom's element follows from how near its
    neighbours are."""
    gen = torch.Generator().manual_seed(seed)
    many = torch.randint(1, 30, (molecules,), generator=gen)
    starts = torch.cat([torch.zeros(1, dtype=torch.long), many.cumsum(0)])
    n = int(starts[-1])
    points = torch.rand(n, 3, generator=gen) * 4
    document = torch.repeat_interleave(torch.arange(molecules), many)
    near = torch.cdist(points, points).masked_fill(document[:, None] != document, 100.).fill_diagonal_(100.).amin(1)
    what = (near * elements / 2).long().clamp(0, elements - 1)
    masked = torch.rand(n, generator=gen) < 1 / 6
    return [t.to(device) for t in (torch.where(masked, elements, what), points, starts.int(), torch.where(masked, what, -1))]


def train(steps=40, molecules=64, elements=16, dtype=torch.float32, seed=0, **kw):
    """Losses of the steps."""
    torch.manual_seed(seed)
    model = Elements(elements, dtype=dtype, **kw)
    opt = gelib.AdamW(model.parameters(), lr=3e-3, weight_decay=1e-3, state_bits=8, seed=seed)
    tokens, points, starts, targets = data(molecules, elements, seed + 1)
    losses = []
    for _ in range(steps):
        opt.zero_grad()
        loss = model(tokens, points, starts, targets).sum() / (targets >= 0).sum().clamp(min=1)
        loss.backward()
        opt.step()
        losses.append(loss.detach())
    return model, [float(v) for v in losses]


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=40)
    ap.add_argument("--bfloat16", action="store_true")
    a = ap.parse_args()
    for k, v in enumerate(train(a.steps, dtype=torch.bfloat16 if a.bfloat16 else torch.float32)[1]):
        if k % 10 == 0 or k == a.steps - 1:
            print("step %d  loss %.5f" % (k, v))
