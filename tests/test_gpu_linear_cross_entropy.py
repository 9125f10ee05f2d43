"""linear_cross_entropy and its gradients against the formulas in float64.  Tolerances, u = 2^-24 and h the half ulp of the type: a logit
is off by (n_in + 4) u of the sum of the moduli of its products; the loss by twice the largest of its row's errors, (classes + 16) u of its sum's
logarithm, and 4 u of what is added.  So a probability is relatively off by twice that error (of the logit and of the log of the sum) and (classes + 16) u; gz = g (p - onehot)
by that of p, by 4 u, and by h where it is rounded for the products; those are sums off by (terms + 8) u of their moduli; results are
rounded once (in check)."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests.test_gpu_group_norm import HALF_ULP, check, u  # noqa: E402


@pytest.fixture(scope="module")
def gelib():
    assert torch.cuda.is_available()
    import gelib_amd
    return gelib_amd


def reference(x, w, b, targets, g, dtype):
    h = 0. if dtype == torch.float32 else HALF_ULP[dtype]
    m, k = x.shape
    n = w.shape[1]
    z = x @ w + b
    ez = ((k + 4) * u * (x.abs() @ w.abs()) + 4 * u * (z.abs() + b.abs())).amax(1, keepdim=True)
    lse = torch.logsumexp(z, 1, keepdim=True)
    there = (targets >= 0)[:, None]
    at = targets.clamp(min=0)[:, None]
    out = {"loss": (torch.where(there, lse - z.gather(1, at), 0.)[:, 0], (2 * ez + (n + 16) * u + 4 * u * (lse.abs() + z.abs().amax(1, keepdim=True)))[:, 0])}
    p = torch.exp(z - lse)
    one = torch.zeros_like(p).scatter_(1, at, 1.)
    gg = torch.where(there, g[:, None], 0.)
    gz = gg * (p - one)
    rel = 2 * ez + (n + 16) * u + 4 * u * (z - lse).abs()
    # float16 values are scaled to below 2^14: the smallest step is 2^-25 / 2^13 of the largest |g|
    least = gg.abs().amax() * 2.0 ** -37 if dtype == torch.float16 else 0.
    egz = gg.abs() * (p * rel + 2.0 ** -126) + 4 * u * gz.abs()
    e16 = egz + h * (gz.abs() + egz) + least * there
    out["gx"] = gz @ w.t(), e16 @ w.abs().t() + (n + 8) * u * (gz.abs() @ w.abs().t())
    out["gw"] = x.t() @ gz, x.abs().t() @ e16 + (m + 8) * u * (x.abs().t() @ gz.abs())
    out["gb"] = gz.sum(0), (egz + (m + 8) * u * gz.abs()).sum(0)
    return out


def case(m, k, n, dtype, seed=0, spread=1.5):
    gen = torch.Generator(device="cuda").manual_seed(m * 7 + k * 3 + n + seed)

    def randn(*s):
        return torch.randn(*s, device="cuda", generator=gen)
    x, w, b = randn(m, k).to(dtype).requires_grad_(), (randn(k, n) * spread / max(k, 1) ** 0.5).to(dtype).requires_grad_(), randn(n).to(dtype).requires_grad_()
    targets = torch.randint(0, n, (m,), device="cuda", generator=gen)
    targets[torch.rand(m, device="cuda", generator=gen) < 0.2] = -100
    return x, w, b, targets, torch.rand(m, device="cuda", generator=gen) + 0.5


# one of everything, sizes around the tiles (16, 64, 128, 256) and their steps, classes of one tile and of many, odd rows that are not aligned
SIZES = [(1, 1, 1), (1, 8, 2), (3, 40, 118), (19, 64, 118), (16, 16, 256), (17, 33, 257), (64, 64, 128), (65, 63, 129), (128, 256, 1000), (129, 72, 513), (300, 1, 5), (257, 130, 384),
         (1000, 8, 40), (5003, 24, 30), (2, 8, 5000), (260, 455, 2052), (7, 0, 6), (40, 24, 36867)]
# long sums of few tiles, which are cut along n_in; the largest that need no matrix cores, and the next
SIZES += [(300, 2048, 118), (70, 4100, 301), (512, 1000, 33), (16, 256, 512), (17, 256, 512), (1, 2048, 1024), (1, 2049, 8), (1024, 64, 32)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_values_and_gradients(gelib, size, dtype):
    x, w, b, targets, g = case(*size, dtype)
    loss = gelib.linear_cross_entropy(x, w, targets, b)
    assert loss.dtype == torch.float32 and loss.shape == targets.shape
    got = dict(zip(("gx", "gw", "gb"), torch.autograd.grad(loss, (x, w, b), g)), loss=loss.detach())
    with torch.no_grad():
        want = reference(x.double(), w.double(), b.double(), targets, g.double(), dtype)
    for name, (v, tol) in want.items():
        check(got[name], v, tol, "%s of %s" % (name, size))
    assert torch.equal(loss, gelib.linear_cross_entropy(x.detach(), w.detach(), targets, b.detach()))
    for t, name in zip(torch.autograd.grad(gelib.linear_cross_entropy(x, w, targets, b), (x, w, b), g), ("gx", "gw", "gb")):
        assert torch.equal(t, got[name])   # fixed orders of summation
    for leaf, name in ((x, "gx"), (w, "gw"), (b, "gb")):
        assert torch.equal(torch.autograd.grad(gelib.linear_cross_entropy(x, w, targets, b), leaf, g)[0], got[name])
    assert torch.equal(gelib.linear_cross_entropy(x, w, targets), gelib.linear_cross_entropy(x, w, targets, torch.zeros_like(b)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_more_classes_than_one_piece(gelib, dtype):
    """The gradient of the logits is formed for some classes after the other where all of them are more than 2^28 bytes."""
    m, k, n = 4099 if dtype == torch.float32 else 8200, 40, 20003
    x, w, b, targets, g = case(m, k, n, dtype)
    assert m * n * x.element_size() > 1 << 28
    loss = gelib.linear_cross_entropy(x, w, targets, b)
    got = dict(zip(("gx", "gw", "gb"), torch.autograd.grad(loss, (x, w, b), g)), loss=loss.detach())
    with torch.no_grad():
        want = reference(x.double(), w.double(), b.double(), targets, g.double(), dtype)
    for name, (v, tol) in want.items():
        check(got[name], v, tol, name)
    for leaf, name in ((x, "gx"), (w, "gw"), (b, "gb")):
        assert torch.equal(torch.autograd.grad(gelib.linear_cross_entropy(x, w, targets, b), leaf, g)[0], got[name])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_many_rows_of_few(gelib, dtype):
    """Long sums over rows, blocks of them for the largest gradient among them (float16); the largest is the last."""
    for size in ((256, 64, 128), (257, 64, 128), (20003, 5, 7), (300001, 8, 9)):
        x, w, b, targets, g = case(*size, dtype)
        targets[-1], g[-1] = 0, 900.
        loss = gelib.linear_cross_entropy(x, w, targets, b)
        got = dict(zip(("gx", "gw", "gb"), torch.autograd.grad(loss, (x, w, b), g)), loss=loss.detach())
        with torch.no_grad():
            want = reference(x.double(), w.double(), b.double(), targets, g.double(), dtype)
        for name, (v, tol) in want.items():
            check(got[name], v, tol, "%s of %s" % (name, size))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_logits_far_apart(gelib, dtype):
    """Logits of hundreds: nothing overflows, a class that has everything leaves the others gradients of zero."""
    x, w, b, targets, g = case(70, 32, 600, dtype, spread=60.)
    loss = gelib.linear_cross_entropy(x, w, targets, b)
    grads = torch.autograd.grad(loss, (x, w, b), g)
    with torch.no_grad():
        want = reference(x.double(), w.double(), b.double(), targets, g.double(), dtype)
    check(loss.detach(), *want["loss"], "loss")
    for t, name in zip(grads, ("gx", "gw", "gb")):
        check(t, *want[name], name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_small_and_large_weights_of_rows(gelib, dtype):
    """Losses averaged over many rows, and scaled up: gradients are those of weight one times the weight, to rounding."""
    x, w, b, targets, _ = case(100, 24, 2000, dtype)
    one = torch.autograd.grad(gelib.linear_cross_entropy(x, w, targets, b), (x, w, b), torch.ones(100, device="cuda"))
    for by in (2.0 ** -20, 2.0 ** 9):
        if dtype == torch.float16 and by < 1:
            continue   # (results themselves are below float16's smallest)
        for t, o in zip(torch.autograd.grad(gelib.linear_cross_entropy(x, w, targets, b), (x, w, b), torch.full((100,), by, device="cuda")), one):
            # (float16: weight one's own smallest step)
            assert ((t.float() - o.float() * by).abs() <= (2.0 ** -25 * by if dtype == torch.float16 else 0.)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_targets_outside(gelib, dtype):
    x, w, b, targets, g = case(40, 24, 50, dtype)
    with torch.no_grad():
        x[4] = float("nan")
    targets[4], targets[7], targets[:3] = -1, -(1 << 60), 5
    loss = gelib.linear_cross_entropy(x, w, targets, b)
    gx, gw, gb = torch.autograd.grad(loss, (x, w, b), g)
    assert torch.isfinite(gw).all() and torch.isfinite(gb).all()
    assert loss[4] == 0 and loss[7] == 0 and torch.isfinite(loss).all()
    assert (gx[4] == 0).all() and (gx[7] == 0).all() and torch.isfinite(gx).all()   # a row left out may hold anything
    with torch.no_grad():
        x[4] = 0
    for bad in (50, 1 << 40):
        targets[2] = bad
        loss = gelib.linear_cross_entropy(x, w, targets, b)
        gx, = torch.autograd.grad(loss, x, g)
        rest = [i for i in range(40) if i != 2]
        assert torch.isnan(loss[2]) and torch.isfinite(loss[rest]).all() and torch.isnan(gx[2]).all() and torch.isfinite(gx[rest]).all()
    targets[:] = -1
    loss = gelib.linear_cross_entropy(x, w, targets, b)
    assert (loss == 0).all() and all((t == 0).all() for t in torch.autograd.grad(loss, (x, w, b), g))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_layouts(gelib, dtype):
    gen = torch.Generator(device="cuda").manual_seed(5)

    def randn(*s):
        return torch.randn(*s, device="cuda", generator=gen).to(dtype)
    big, W = randn(6, 9, 80), randn(100, 70)
    for x in (big, big[:, :, 5:37], big[:, 2:7, 8:24], big.transpose(0, 1), big[..., ::2], big[0, 0], big[:1, :1, :16].expand(3, 5, 16)):
        for w in (W[:x.shape[-1], :48], W[1:1 + x.shape[-1], 3:36], randn(40, 80)[:, :x.shape[-1]].t()):
            targets = torch.randint(-1, w.shape[1], (*x.shape[:-1], 2), device="cuda", generator=gen)[..., 0]
            outs = []
            for f in (lambda t: t, lambda t: t.contiguous()):
                ts = [f(t).detach().requires_grad_() for t in (x, w)]
                loss = gelib.linear_cross_entropy(ts[0], ts[1], f(targets))
                outs.append((loss, *torch.autograd.grad(loss, ts, torch.ones((), device="cuda").expand(loss.shape))))
            for a, b in zip(*outs):
                assert torch.equal(a, b)


def test_against_differences_and_twice(gelib):
    """Central differences over 2^-7: 1 % of the gradient's norm (third derivatives, rounding)."""
    x, w, b, targets, g = case(30, 12, 20, torch.float32)
    ts = [x, w, b]
    gen = torch.Generator(device="cuda").manual_seed(2)

    def f(x, w, b):
        return (gelib.linear_cross_entropy(x, w, targets, b).double() * g.double()).sum()
    grads = torch.autograd.grad(f(*ts), ts)
    graph = torch.autograd.grad(f(*ts), ts, create_graph=True)
    for a, c in zip(grads, graph):
        assert torch.allclose(a, c, rtol=1e-4, atol=1e-5)
    ds = [torch.randn(t.shape, device="cuda", generator=gen) for t in ts]
    second = torch.autograd.grad(sum((a * d).sum() for a, d in zip(graph, ds)), ts)
    for i, t in enumerate(ts):
        d = torch.randn(t.shape, device="cuda", generator=gen)
        d /= d.norm()
        near = [[(s + e * d).detach().requires_grad_() if j == i else s for j, s in enumerate(ts)] for e in (2.0 ** -7, -2.0 ** -7)]
        slope = (f(*near[0]) - f(*near[1])).detach() / 2.0 ** -6
        assert abs(float(slope - (grads[i].double() * d).sum())) <= 1e-2 * float(grads[i].norm()) + 1e-3
        plus, minus = (sum((a.double() * c.double()).sum() for a, c in zip(torch.autograd.grad(f(*n), n), ds)) for n in near)
        assert abs(float((plus - minus) / 2.0 ** -6 - (second[i].double() * d).sum())) <= 2e-2 * float(second[i].norm()) + 5e-3


def test_another_stream_and_graph(gelib):
    x, w, b, targets, g = case(300, 200, 900, torch.bfloat16)
    ts = (x, w, b)

    def step():
        y = gelib.linear_cross_entropy(x, w, targets, b)
        return (y.detach(), *torch.autograd.grad(y, ts, g))   # (no graph outlives a step: its nodes belong to the stream that it was made on)
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, c in zip(got, want):
        assert torch.equal(a, c)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(300, 200, device="cuda"))
            targets.copy_(torch.randint(-1, 900, (300,), device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in out]
        for a, c in zip(kept, step()):
            assert torch.equal(a, c)


def test_nothing(gelib):
    x, w, b = torch.randn(0, 8, device="cuda", requires_grad=True), torch.randn(8, 5, device="cuda", requires_grad=True), torch.randn(5, device="cuda", requires_grad=True)
    loss = gelib.linear_cross_entropy(x, w, torch.empty(0, device="cuda", dtype=torch.long), b)
    assert loss.shape == (0,)
    gx, gw, gb = torch.autograd.grad(loss, (x, w, b), loss)
    assert gx.shape == x.shape and (gw == 0).all() and (gb == 0).all()


def test_refusals(gelib):
    x, w, b, t = torch.randn(4, 8, device="cuda"), torch.randn(8, 6, device="cuda"), torch.randn(6, device="cuda"), torch.zeros(4, device="cuda", dtype=torch.long)
    f = gelib.linear_cross_entropy
    for bad, error in ((lambda: f(x, w[:7], t), ValueError), (lambda: f(x, w[0], t), ValueError), (lambda: f(x, w[:, :0], t), ValueError), (lambda: f(x.cpu(), w, t), ValueError),
                       (lambda: f(x, w.cpu(), t), ValueError), (lambda: f(x.half(), w, t), TypeError), (lambda: f(x.double(), w.double(), t), TypeError), (lambda: f(x, w, t.int()), TypeError),
                       (lambda: f(x, w, t[:3]), ValueError), (lambda: f(x, w, t.cpu()), ValueError), (lambda: f(x, w, t, b[:5]), ValueError), (lambda: f(x, w, t, b.half()), TypeError)):
        with pytest.raises(error):
            bad()
