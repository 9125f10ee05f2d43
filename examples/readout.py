"""A network on invariants behind an equivariant layer, trained with the operators on real channels:

    SO3vecs x, y  ->  CGproduct_linear (one complex matrix per l)  ->  norms of the parts, one a channel and l (invariants)
                  ->  residual blocks: u + linear_act(group_norm_act(u))  ->  a number a sample

The cells of a sample (the atoms of a molecule, padded to the largest) are positions of the norm, their number is its length.  All
weights, the complex matrices among them, are changed by one AdamW step.

    python examples/readout.py [--steps 60] [--bits 8]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import gelib_amd as gelib  # noqa: E402


class Readout(torch.nn.Module):

    def __init__(self, maxl, tau, width, blocks=2, dtype=torch.float32, device="cuda"):
        super().__init__()
        self.maxl, self.dtype = maxl, dtype
        t = {l: tau for l in range(maxl + 1)}
        from gelib_amd import cabi
        taus = cabi.so3type_product(t, t, maxl)

        def real(*shape, scale=0.0, at=0.0):
            return torch.nn.Parameter((at + scale * torch.randn(*shape, device=device)).to(dtype))
        self.W = torch.nn.ParameterList([torch.nn.Parameter(torch.randn(taus[l], tau, dtype=torch.complex64, device=device) / taus[l] ** 0.5)
                                         for l in range(maxl + 1)])
        n = (maxl + 1) * tau
        self.first, self.first_bias = real(n, width, scale=n ** -0.5), real(width)
        self.gain = torch.nn.ParameterList([real(width, at=1.0) for _ in range(blocks)])
        self.shift = torch.nn.ParameterList([real(width) for _ in range(blocks)])
        self.matrix = torch.nn.ParameterList([real(width, width, scale=width ** -0.5) for _ in range(blocks)])
        self.bias = torch.nn.ParameterList([real(width) for _ in range(blocks)])
        self.last = real(width, 8, scale=width ** -0.5)   # (eight numbers a sample: their mean is the answer)

    def forward(self, x, y, lengths):
        """x, y: SO3vecs with parts (samples * cells, 2l+1, tau); lengths: int32, the cells of each sample that exist."""
        v = gelib.CGproduct_linear(x, y, gelib.SO3weights(*self.W), self.maxl)
        parts = [p.as_subclass(torch.Tensor) for p in v.parts.values()]
        # squared norms do not change when a vector is rotated
        u = torch.cat([torch.log1p((p.real.square() + p.imag.square()).sum(1)) for p in parts], 1).to(self.dtype)
        u = gelib.linear_act(u.view(len(lengths), -1, u.shape[1]), self.first, self.first_bias, act="silu")
        groups = max(1, u.shape[-1] // 16)
        for gain, shift, matrix, bias in zip(self.gain, self.shift, self.matrix, self.bias):
            h = gelib.group_norm_act(u, groups, gain, shift, act="silu", lengths=lengths)
            u = gelib.linear_act(h, matrix, bias, residual=u, act="gelu")
        u = gelib.linear_act(u, self.last)
        live = torch.arange(u.shape[1], device=u.device) < lengths[:, None]
        return (u.float().mean(2) * live).sum(1) / lengths.clamp(min=1)


def data(samples, cells, maxl, tau, seed, device="cuda"):
    """Random vectors, how many cells of each sample exist, and an invariant of them to learn."""
    gen = torch.Generator(device=device).manual_seed(seed)

    def vec():
        return gelib.SO3vec(*[torch.view_as_complex(torch.randn(samples * cells, 2 * l + 1, tau, 2, device=device, generator=gen)) for l in range(maxl + 1)])
    x, y = vec(), vec()
    lengths = torch.randint(1, cells + 1, (samples,), device=device, generator=gen, dtype=torch.int32)
    dots = sum((a.as_subclass(torch.Tensor).conj() * b.as_subclass(torch.Tensor)).sum((1, 2)).real for a, b in zip(x.parts.values(), y.parts.values()))
    live = torch.arange(cells, device=device) < lengths[:, None]
    target = (torch.tanh(0.1 * dots).view(samples, cells).square() * live).sum(1) / lengths
    return x, y, lengths, target


def train(steps=60, bits=8, samples=64, cells=12, maxl=2, tau=4, width=64, dtype=torch.float32, seed=0):
    """Losses of the steps."""
    torch.manual_seed(seed)
    model = Readout(maxl, tau, width, dtype=dtype)
    opt = gelib.AdamW(model.parameters(), lr=3e-3, weight_decay=1e-3, state_bits=bits, seed=seed)
    x, y, lengths, target = data(samples, cells, maxl, tau, seed + 1)
    losses = []
    for _ in range(steps):
        opt.zero_grad()
        loss = (model(x, y, lengths) - target).square().mean()
        loss.backward()
        opt.step()
        losses.append(loss.detach())
    return model, [float(v) for v in losses]


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--bits", type=int, choices=(8, 32), default=8)
    a = ap.parse_args()
    for k, v in enumerate(train(a.steps, a.bits)[1]):
        if k % 10 == 0 or k == a.steps - 1:
            print("step %d  loss %.5f" % (k, v))
