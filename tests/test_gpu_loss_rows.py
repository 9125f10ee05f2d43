"""linear_cross_entropy at the ends of what floats hold, in every way that the kernels take (without matrix cores, logits in pieces of n_in, tiles,
some classes after the other)."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

u = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
# rows, n_in, classes: without matrix cores; tiles; few rows with long sums (both products in pieces); widths that no wide load takes; many classes
SIZES = [(9, 8, 20), (300, 64, 118), (300, 5000, 118), (257, 63, 129), (1500, 16, 1000)]


@pytest.fixture(scope="module")
def gelib():
    assert torch.cuda.is_available()
    import gelib_amd
    return gelib_amd


def left_out(gelib, m, k, n, dtype):
    gen = torch.Generator(device="cuda").manual_seed(m + k)
    x, w = torch.randn(m, k, device="cuda", generator=gen).to(dtype), (torch.randn(k, n, device="cuda", generator=gen) / k ** 0.5).to(dtype)
    w[k // 2, n // 2], w[0, n - 1] = float("inf"), float("nan")
    targets = torch.randint(0, n, (m,), device="cuda", generator=gen)
    out = torch.rand(m, device="cuda", generator=gen) < 0.5
    out[0], out[-1] = True, True
    targets[out] = -1
    x.requires_grad_(), w.requires_grad_()
    loss = gelib.linear_cross_entropy(x, w, targets)
    gx, = torch.autograd.grad(loss, x, torch.ones_like(loss))
    assert (loss[out] == 0).all() and (gx[out] == 0).all() and torch.isnan(gx[~out]).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_rows_left_out_beside_infinite_weights(gelib, size, dtype):
    left_out(gelib, *size, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_rows_left_out_of_more_classes_than_one_piece(gelib, dtype):
    for k in (40, 41):
        left_out(gelib, 4099 if dtype == torch.float32 else 8200, k, 20003, dtype)


FAR = [(9, 8, 25), (300, 64, 124), (300, 5000, 124), (1500, 16, 1026)]   # (classes whose log is nearly a multiple of 2^-8)


def far_logits(n):
    """Whole numbers B from 40000 to 65000, where float32's step is 2^-8 and B + log n a multiple of it to a tenth of half a step (that is up to
    n), while the product of B, or of that, with log2(e) is as far from float32 numbers as can be."""
    step = 2.0 ** -8

    def off(v, step):   # in half steps
        return abs(v / step - round(v / step)) * 2
    assert off(math.log(n), step) < 0.1
    log2e = float(torch.tensor(1.4426950408889634, dtype=torch.float32))
    found = [], []
    for i in range(40000, 65000):
        for v, to in zip((i, round((i + math.log(n)) / step) * step), found):
            if off(v * log2e, 2 * step if v * log2e >= 65536 else step) > 0.95:
                to.append(float(i))
    return found[0][::len(found[0]) // 3] + found[1][::len(found[1]) // 3]


@pytest.mark.parametrize("size", FAR, ids=lambda s: "x".join(map(str, s)))
def test_logits_far_from_zero(gelib, size):
    """Equal logits, float32 numbers: log n of loss and probabilities of 1 / n, whatever the logits are.  Tolerance: log of the sum is a float32 number
    a twentieth of its last place (2^-8) from the truth, and its own logarithm, exponentials and sums are off by (n + 16) u."""
    m, k, n = size
    for B in far_logits(n):
        x, w = torch.zeros(m, k, device="cuda"), torch.zeros(k, n, device="cuda")
        b = torch.full((n,), B, device="cuda", requires_grad=True)
        targets = torch.zeros(m, device="cuda", dtype=torch.long)
        loss = gelib.linear_cross_entropy(x, w, targets, b)
        gb, = torch.autograd.grad(loss.sum(), b)
        tol = 2.0 ** -8 / 20 + (n + 16) * u
        assert ((loss.double() - math.log(n)).abs() <= tol).all(), B
        assert ((gb[1:].double() * n / m - 1).abs() <= tol + (m + 16) * u).all(), B


@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_infinite_logits(gelib, size):
    """log of a sum with an infinite term is infinite: so is the loss of the other classes, and the loss of that class is none (infinity less infinity).
    -infinity is a class without a share; where all are, there is no loss to speak of (NaN), in that row only."""
    m, k, n = size
    gen = torch.Generator(device="cuda").manual_seed(m)
    x, w = torch.randn(m, k, device="cuda", generator=gen), torch.randn(k, n, device="cuda", generator=gen) / k ** 0.5
    targets = torch.arange(m, device="cuda") % n
    for at in (0, n // 2, n - 1):
        b = torch.randn(n, device="cuda", generator=gen)
        b[at] = float("inf")
        loss = gelib.linear_cross_entropy(x, w, targets, b)
        assert torch.isnan(loss[targets == at]).all() and (loss[targets != at] == float("inf")).all()
        b[at] = float("-inf")
        loss = gelib.linear_cross_entropy(x, w, targets, b)
        keep = torch.arange(n, device="cuda") != at
        other = gelib.linear_cross_entropy(x, w[:, keep].contiguous(), (targets - (targets > at).long()).clamp(max=n - 2), b[keep])
        seen = targets != at
        assert (loss[~seen] == float("inf")).all() and torch.allclose(loss[seen], other[seen], rtol=1e-5, atol=1e-5)
    loss = gelib.linear_cross_entropy(x, w, targets, torch.full((n,), float("-inf"), device="cuda"))
    assert torch.isnan(loss).all()
