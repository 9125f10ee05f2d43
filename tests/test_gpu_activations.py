"""The activations of float32 layers against float64, over values as norms give them.  Tolerance: both this form and torch's float32
operations are a handful of roundings, each of about half a unit of the value, so their root mean squares are alike: 1.2 times for the
values, whose last rounding is the largest; 1.7 for the slopes, a sum of terms that carry the exponential's roundings twice."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("by", ["linear", "norm"])
def test_as_exact_as_torchs_float32_operations(by, act):
    import gelib_amd as gelib
    f = getattr(torch.nn.functional, act)
    gen = torch.Generator(device="cuda").manual_seed(1)
    if by == "linear":
        z = torch.randn(1 << 19, 1, device="cuda", generator=gen)
        w = torch.ones(1, 1, device="cuda")
        x = z.clone().requires_grad_()
        y = gelib.linear_act(x, w, act=act)
    else:   # groups of -1 and 1 are their own norms, weight and bias make them z
        n = 1 << 19
        w, x = torch.randn(n, device="cuda", generator=gen), torch.randn(n, device="cuda", generator=gen).requires_grad_()
        ones = torch.ones(1, 2, n, device="cuda")
        ones[0, 1] = -1
        y = gelib.group_norm_act(ones, n, w, x, eps=0.0, act=act)[0, 0]
        z = w + x.detach()
    slope, = torch.autograd.grad(y.sum(), x)
    outs = []
    for t in (z, z.double()):
        t = t.clone().requires_grad_()
        v = f(t)
        outs.append((v.detach().double(), torch.autograd.grad(v.sum(), t)[0].double()))
    for name, got, times in (("value", y, 1.2), ("slope", slope, 1.7)):
        k = name == "slope"
        ours, plain = ((a.detach().double().view(-1) - outs[1][k].view(-1)).square().mean().sqrt() for a in (got, outs[0][k]))
        assert ours <= times * plain, (name, float(ours / plain))


def test_sums_over_many_samples():
    """The gradient of a norm's bias over 32768 samples is as far from float64 as torch's float32 sum of as many terms (1.3 times: both add in short
    chains, of a term's rounding each)."""
    import gelib_amd as gelib
    gen = torch.Generator(device="cuda").manual_seed(2)
    x, g = (torch.randn(32768, 1, 64, device="cuda", generator=gen) for _ in range(2))
    b = torch.zeros(64, device="cuda", requires_grad=True)
    got, = torch.autograd.grad(gelib.group_norm_act(x, 8, None, b), b, g)
    want = g.double().sum((0, 1))
    ours, plain = ((t.double() - want).square().mean().sqrt() for t in (got, g.sum((0, 1))))
    assert ours <= 1.3 * plain + 2.0 ** -24 * want.abs().max(), (float(ours), float(plain))
