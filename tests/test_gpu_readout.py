"""The operators on real channels together, behind an equivariant layer (examples/readout.py): the network's answer is that of torch's
operations and does not change when its vectors are rotated, and training it changes all weights and brings the loss down."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def readout():
    assert torch.cuda.is_available()
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "readout.py")
    spec = importlib.util.spec_from_file_location("readout", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def plain(model, x, y, lengths):
    """The same network from torch's operations, behind the same product."""
    import gelib_amd as gelib
    F = torch.nn.functional
    v = gelib.CGproduct_linear(x, y, gelib.SO3weights(*model.W), model.maxl)
    u = torch.cat([torch.log1p((p.as_subclass(torch.Tensor).abs() ** 2).sum(1)) for p in v.parts.values()], 1)
    u = F.silu(u.view(len(lengths), -1, u.shape[1]) @ model.first + model.first_bias)
    for gain, shift, matrix, bias in zip(model.gain, model.shift, model.matrix, model.bias):
        h = torch.zeros_like(u)
        for n, k in enumerate(lengths.tolist()):
            h[n, :k] = F.silu(F.group_norm(u[n:n + 1, :k].transpose(1, 2), max(1, u.shape[-1] // 16), gain, shift).transpose(1, 2))[0]
        u = F.gelu(h @ matrix + bias) + u
    u = (u @ model.last).mean(2)
    return torch.stack([u[n, :k].mean() for n, k in enumerate(lengths.tolist())])


def test_same_as_torch(readout):
    torch.manual_seed(3)
    model = readout.Readout(2, 4, 48)
    x, y, lengths, target = readout.data(9, 7, 2, 4, 5)
    got, want = model(x, y, lengths), plain(model, x, y, lengths)
    assert torch.allclose(got, want, rtol=1e-4, atol=1e-5)
    a = torch.autograd.grad((got - target).square().sum(), list(model.parameters()))
    b = torch.autograd.grad((want - target).square().sum(), list(model.parameters()))
    for p, q in zip(a, b):
        assert (p - q).abs().max() <= 1e-3 * q.abs().max() + 1e-6


def test_invariant(readout):
    """Rotated by 0.7 about the polar axis: element m of a part turns by exp(-i m 0.7)."""
    import gelib_amd as gelib
    torch.manual_seed(3)
    model = readout.Readout(2, 4, 64)
    x, y, lengths, _ = readout.data(16, 5, 2, 4, 6)

    def turned(v):
        out = []
        for l, p in v.parts.items():
            m = torch.arange(-l, l + 1, device="cuda")
            out.append(p.as_subclass(torch.Tensor) * torch.polar(torch.ones_like(m, dtype=torch.float32), -0.7 * m)[:, None])
        return gelib.SO3vec(*out)
    with torch.no_grad():
        a, b = model(x, y, lengths), model(turned(x), turned(y), lengths)
    assert torch.allclose(a, b, rtol=1e-4, atol=1e-5) and a.std() > 1e-3


@pytest.mark.parametrize("bits,dtype", [(32, torch.float32), (8, torch.float32), (8, torch.bfloat16)], ids=str)
def test_training(readout, bits, dtype):
    torch.manual_seed(0)
    before = [p.detach().clone() for p in readout.Readout(2, 4, 64, dtype=dtype).parameters()]
    model, losses = readout.train(steps=60, bits=bits, dtype=dtype)
    assert all(torch.isfinite(p).all() for p in model.parameters())
    assert all(not torch.equal(p, q) for p, q in zip(model.parameters(), before))
    assert losses[-1] < 0.3 * losses[0], losses
    assert readout.train(steps=3, bits=bits, dtype=dtype)[1] == readout.train(steps=3, bits=bits, dtype=dtype)[1]   # runs repeat
