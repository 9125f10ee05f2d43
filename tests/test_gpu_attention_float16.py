"""Attention's weights and their gradients in float16, whose least normal value is 2^-14: both are brought into its range by powers of two
for the products that take them as float16 values.  Formulas in float64; tolerances, u = 2^-24, h = 2^-11: as in test_gpu_attention.py, but that
what the smallest steps cost is
  weights of the values, which stand at 2^7 and more for a row's largest:  2^-25 / 2^7 = 2^-32 of the row's largest weight;
  weights of the values' gradients, times 2^12:                            2^-37;
  gradients of scores, which stand at 2^11 and more for the largest of a query (gq) or of a key (gk):  2^-25 / 2^11 = 2^-36 of that."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests.test_gpu_group_norm import check, u  # noqa: E402

H = 2.0 ** -11


@pytest.fixture(scope="module")
def gelib():
    assert torch.cuda.is_available()
    import gelib_amd
    return gelib_amd


def reference(q, k, v, g, scale, x=None, xk=None, slopes=None):
    """{name: (value, tolerance)}; q, g (nq, heads, dim), k, v (nk, kv heads, dim), float64"""
    nq, heads, dim = q.shape
    nk, kv = k.shape[:2]
    kk, vv = (t.repeat_interleave(heads // kv, 1).transpose(0, 1) for t in (k, v))
    qq, gg = q.transpose(0, 1), g.transpose(0, 1)
    s = scale * qq @ kk.transpose(1, 2)
    es = abs(scale) * (dim + 4) * u * (qq.abs() @ kk.abs().transpose(1, 2))
    if x is not None:
        apart = x[:, None] - xk[None]
        far = apart.square().sum(2).sqrt()
        s = s - slopes[:, None, None] * far
        es = es + 8 * u * slopes.abs()[:, None, None] * far
    es = es + 4 * u * s.abs()
    p = torch.softmax(s, 2)
    rel = 2 * es.amax(2, keepdim=True) + (nk + 16) * u
    top = p.amax(2, keepdim=True)
    y = p @ vv
    ey = (p * (rel + H) + 2.0 ** -32 * top) @ vv.abs() + (nk + 8) * u * (p @ vv.abs())
    out = {"y": (y.transpose(0, 1), ey.transpose(0, 1))}
    dp = gg @ vv.transpose(1, 2)
    edp = (dim + 4) * u * (gg.abs() @ vv.abs().transpose(1, 2))
    D = (gg * y).sum(2, keepdim=True)
    # D from the rounded y is mended by the sum of ds, to the errors of p and of gy . v
    eD = (p * (rel * (dp - D).abs() + edp)).sum(2, keepdim=True) + (nk + dim) * u * (p * dp.abs()).sum(2, keepdim=True) + (dim + 4) * u * (gg * y).abs().sum(2, keepdim=True)
    ds = p * (dp - D)
    eds = p * rel * (dp - D).abs() + p * (edp + eD) + 4 * u * ds.abs()

    def e16(over):   # rounded to float16, of the largest along `over`
        return eds + H * (ds.abs() + eds) + 2.0 ** -36 * (ds.abs() + eds).amax(over, keepdim=True)
    # (gq: D's own error comes back through sums with rounded p)
    lack = (H * y.abs() * gg.abs()).sum(2, keepdim=True) + (ey * gg.abs()).sum(2, keepdim=True)
    out["gq"] = ((scale * ds @ kk).transpose(0, 1),
                 (abs(scale) * (e16(2) + (nk + 8) * u * ds.abs() + lack * (p * (rel + 2 * H) + 2.0 ** -37)) @ kk.abs()).transpose(0, 1))

    def group(t):
        return t.unflatten(0, (kv, heads // kv)).sum(1).transpose(0, 1)
    terms = nq * heads // kv + 8
    out["gk"] = group(scale * ds.transpose(1, 2) @ qq), group(abs(scale) * (e16(1) + terms * u * ds.abs()).transpose(1, 2) @ qq.abs())
    out["gv"] = group(p.transpose(1, 2) @ gg), group((p * (rel + H + terms * u) + 2.0 ** -37).transpose(1, 2) @ gg.abs())
    if x is not None:
        out["gslopes"] = -(ds * far).sum((1, 2)), ((eds + (nk + nq + 32) * u * ds.abs()) * far).sum((1, 2))
    return out


def compare(gelib, nq, nk, heads, kv, dim, weight, points=False, q_scale=1.0, v_scale=1.0, seed=0, scale=None):
    gen = torch.Generator(device="cuda").manual_seed(seed + nq + nk + dim)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)
    q, k, v, g = (randn(nq, heads, dim) * q_scale).half(), randn(nk, kv, dim).half(), (randn(nk, kv, dim) * v_scale).half(), (randn(nq, heads, dim).clamp(-4, 4) * weight).half()
    x = xk = slopes = None
    leaves = {"gq": q, "gk": k, "gv": v}
    if points:
        x, xk, slopes = randn(nq, 3) * 2, randn(nk, 3) * 2, torch.rand(heads, device="cuda", generator=gen) + 0.05
        leaves["gslopes"] = slopes
    for t in leaves.values():
        t.requires_grad_()
    y = gelib.attention(q[None], k[None], v[None], None if x is None else x[None], slopes, key_points=None if x is None else xk[None], scale=scale)[0]
    got = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), g)), y=y.detach())
    with torch.no_grad():
        want = reference(q.double(), k.double(), v.double(), g.double(), dim ** -0.5 if scale is None else scale, *(t.double() if t is not None else None for t in (x, xk, slopes)))
    for name, (value, tol) in want.items():
        assert got[name].dtype == torch.float32 or (value.abs() + tol).max() < 65504, name
        check(got[name], value, tol, "%s of %s x %s, weight %s" % (name, nq, nk, weight))


# a block's worth, a wave's, single queries and few keys (pieces)
SIZES = [(130, 2048, 2, 1, 64), (20, 33, 4, 2, 32), (1, 3000, 4, 2, 64), (700, 5, 2, 2, 16), (64, 600, 2, 2, 128)]


@pytest.mark.parametrize("points", [False, True], ids=["plain", "points"])
@pytest.mark.parametrize("weight", [2.0 ** -10, 2.0 ** -14, 1.0, 2.0 ** 10, 2.0 ** 13])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_small_and_large_gradients(gelib, size, weight, points):
    """Losses averaged over many points, and scaled up.  (Not asked for: results that float16 does not hold.)"""
    if size[0] > 200:
        weight = min(weight, 2.0 ** 8)
    compare(gelib, *size, weight, points, v_scale=1.0 if weight < 100 else 2.0 ** -8)


@pytest.mark.parametrize("points", [False, True], ids=["plain", "points"])
def test_gradients_of_scores_beyond_float16(gelib, points):
    """Gradients of scores of 1e5 to 1e6 whose products are within float16."""
    for size in ((3, 4, 2, 2, 64), (1, 900, 2, 1, 64), (100, 100, 2, 1, 64)):
        compare(gelib, *size, 4096.0, points, q_scale=4.0 ** -1, v_scale=8.0, scale=2.0 ** -8)


def test_rows_of_unlike_weights(gelib):
    """Gradients that differ by 2^20 from one query to the next, the large ones first, last, and in between: each query's own are as exact as alone."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    nq, nk, dim = 160, 400, 32
    q, k, v = (torch.randn(n, 2, dim, device="cuda", generator=gen).half() for n in (nq, nk, nk))
    q /= 32   # (so that gq, scale ds k, stays in the range of float16's normal values)
    for t in (q, k, v):
        t.requires_grad_()
    for order in (1, -1, 0):
        e = torch.linspace(-10, 10, nq, device="cuda") if order else torch.rand(nq, device="cuda", generator=gen) * 20 - 10
        g = (torch.randn(nq, 2, dim, device="cuda", generator=gen) * torch.exp2(e * (order or 1))[:, None, None]).half()
        y = gelib.attention(q[None], k[None], v[None], scale=8.0)[0]
        got = dict(zip(("gq", "gk", "gv"), torch.autograd.grad(y, (q, k, v), g)))
        with torch.no_grad():
            want = reference(q.double(), k.double(), v.double(), g.double(), 8.0)
        for name, t in got.items():
            check(t, *want[name], "%s, order %s" % (name, order))


def test_many_keys(gelib):
    """65536 keys under a few queries: weights of 2^-16, far below float16's normal values, gradients of the values that are not."""
    for nq in (1, 3):
        compare(gelib, nq, 65536, 2, 1, 32, 2.0 ** 12, q_scale=0.25, v_scale=2.0 ** -6)


def test_many_small_weights_beside_a_large_one(gelib):
    """One key has nearly everything, 65535 others 2^-26 each, 2^-10 together: all that is in y when the one's value is zero.  (So many samples, of the same
    keys, that none is cut into pieces.)"""
    nk, dim, n = 65536, 16, 2048
    q, k, v = torch.zeros(1, 1, dim, device="cuda"), torch.zeros(nk, 1, dim, device="cuda"), torch.ones(nk, 1, dim, device="cuda")
    q[:, :, 0] = 1
    k[1:, :, 0] = -18.03
    v[0] = 0
    q, k, v = q.half(), k.half(), v.half()
    y = gelib.attention(*(t.expand(n, *t.shape) for t in (q, k, v)), scale=1.0)
    want = reference(q.double(), k.double(), v.double(), torch.zeros_like(q).double(), 1.0)["y"]
    check(y, *(t.expand(n, *t.shape) for t in want), "y")


@pytest.mark.parametrize("size", [(300, 3, 8, 8, 32), (100, 7, 8, 4, 16), (64, 24, 8, 8, 32)], ids=lambda s: "x".join(map(str, s)))
def test_gradients_of_points_are_float32(gelib, size):
    """What float16 operands do not round: relative errors of the whole gradients of points and slopes.  An exponent, below 4 in log2 units, is
    rounded by at most 2^-23 (1.4 u of a weight), hardware's exponential by 2 u, distance, gy . v - D and the product by 2 u each at the
    most, independently: 4 u is more than the root of the sum of their squares.  Gradients of slopes: a row's ds sum to zero, so the sum of ds
    times distances that are nearly alike is small beside its terms; it is off by 4 u of their moduli, and so are the rows, independently."""
    n, m, heads, kv, dim = size
    gen = torch.Generator(device="cuda").manual_seed(n)
    q, k, v, g = ((torch.randn(n, m, h, dim, device="cuda", generator=gen)).half() for h in (heads, kv, kv, heads))
    x, s = (torch.rand(n, m, 3, device="cuda", generator=gen) * 6).requires_grad_(), (torch.rand(heads, device="cuda", generator=gen) + 0.1).requires_grad_()
    got = torch.autograd.grad(gelib.attention(q, k, v, x, s), (x, s), g)
    X, S = (t.detach().double().requires_grad_() for t in (x, s))
    kk, vv = (t.double().repeat_interleave(heads // kv, 2).transpose(1, 2).contiguous() for t in (k, v))
    sq = (X[:, :, None] - X[:, None]).square().sum(3)
    same = torch.eye(m, dtype=torch.bool, device="cuda")
    far = sq.masked_fill(same, 1.).sqrt().masked_fill(same, 0.)
    p = torch.softmax(q.double().transpose(1, 2).contiguous() @ kk.transpose(2, 3).contiguous() * dim ** -0.5 - S.view(1, -1, 1, 1) * far[:, None], 3)
    want = torch.autograd.grad((p @ vv).transpose(1, 2), (X, S), g.double(), retain_graph=True)
    with torch.no_grad():
        dp = g.double().transpose(1, 2).contiguous() @ vv.transpose(2, 3).contiguous()
        ds = p * (dp - (p * dp).sum(3, keepdim=True))
        rows = (ds.abs() * far[:, None]).sum(3).square().sum((0, 2)).sqrt()
    assert (got[0].double() - want[0]).norm() <= 4 * u * want[0].norm()
    assert ((got[1].double() - want[1]).abs() <= 4 * u * rows + u * want[1].abs()).all()


@pytest.mark.parametrize("size", [(40, 100, 2, 2, 32), (150, 200, 4, 2, 64), (150, 700, 8, 2, 64)], ids=lambda s: "x".join(map(str, s)))
def test_gradients_of_infinity_stay_where_they_are(gelib, size):
    """A gradient that overflowed (what a scaled loss is watched for): gq of the other queries and heads has the bits that it has without it."""
    nq, nk, heads, kv, dim = size
    gen = torch.Generator(device="cuda").manual_seed(nq)
    q, k, v, g = (torch.randn(1, n, h, dim, device="cuda", generator=gen).half() for n, h in ((nq, heads), (nk, kv), (nk, kv), (nq, heads)))
    x, xk, s = torch.randn(1, nq, 3, device="cuda", generator=gen), torch.randn(1, nk, 3, device="cuda", generator=gen), torch.rand(heads, device="cuda", generator=gen).requires_grad_()
    leaves = [t.requires_grad_() for t in (q, k, v)]

    def grads(g):
        return torch.autograd.grad(gelib.attention(q, k, v, x, s, key_points=xk), [*leaves, s], g)
    want = grads(g)
    bad = g.clone()
    bad[0, 7, 1, 3] = float("inf")
    got = grads(bad)
    other = torch.ones(1, nq, heads, dtype=torch.bool, device="cuda")
    other[0, 7, 1] = False
    assert torch.equal(got[0][other], want[0][other]) and not torch.isfinite(got[0][~other]).all()
    rest = [h for h in range(kv) if h != 1 // (heads // kv)]
    assert torch.equal(got[1][:, :, rest], want[1][:, :, rest]) and torch.equal(got[2][:, :, rest], want[2][:, :, rest])
    assert torch.equal(got[3][torch.arange(heads) != 1], want[3][torch.arange(heads) != 1])


def test_recorded(gelib):
    """Powers of two are chosen anew at every replay: gradients that grow and shrink by 2^8 between them."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    q, k, v = (torch.randn(2, 90, h, 32, device="cuda", generator=gen).half().requires_grad_() for h in (4, 2, 2))
    g = torch.randn(2, 90, 4, 32, device="cuda", generator=gen).half()

    def step():
        y = gelib.attention(q, k, v)
        return (y.detach(), *torch.autograd.grad(y, (q, k, v), g))   # (no graph outlives a step)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for e in (0, -8, 8, 0):
        g.copy_(torch.randn(2, 90, 4, 32, device="cuda", generator=gen) * 2.0 ** e)
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in out]
        for a, b in zip(kept, step()):
            assert torch.equal(a, b)
