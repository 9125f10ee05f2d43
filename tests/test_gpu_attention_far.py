"""Attention where the keys that come first have no share: scores of -infinity, or so far below the others that their weights are zero.  The rest
of the document then has to come out as if it stood alone.  References and tolerances: test_gpu_attention.py's, of the keys that have a
share; the others add terms of weight exp(-1000) and less, which are zero in float64 as in float32."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests.test_gpu_attention import TYPES, document  # noqa: E402
from tests.test_gpu_group_norm import check  # noqa: E402


@pytest.fixture(scope="module")
def gelib():
    assert torch.cuda.is_available()
    import gelib_amd
    return gelib_amd


# keys before the others: a tile (of 64 or 32), two, and many (cut into pieces where queries are few)
FIRST = [64, 128, 1500]
# queries and the keys that have a share: short documents (a wave a block), single queries (pieces), long ones
OTHERS = [(5, 7), (1, 40), (150, 90)]
# how far those lie from the queries: scores near zero, and ones whose exponentials are small or nothing in float32
AWAY = [0., 40., 200.]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("first", FIRST)
@pytest.mark.parametrize("nq,nk", OTHERS, ids=lambda v: str(v))
@pytest.mark.parametrize("dim", [16, 64, 128])
def test_scores_of_minus_infinity(gelib, dim, nq, nk, first, dtype):
    """Keys of -infinity in the one channel that queries look at.  (Gradients of such queries are 0 times infinity: not compared.)"""
    gen = torch.Generator(device="cuda").manual_seed(first + nq + dim)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen).to(dtype)
    for away in AWAY:
        q, k, v, g = torch.zeros(nq, 4, dim, device="cuda", dtype=dtype), randn(first + nk, 2, dim), randn(first + nk, 2, dim), randn(nq, 4, dim)
        q[:, :, 0] = 1
        k[:, :, 0] -= away
        k[:first, :, 0] = float("-inf")
        k.requires_grad_(), v.requires_grad_()
        y = gelib.attention(q[None], k[None], v[None], scale=1.0)[0]
        gk, gv = torch.autograd.grad(y, (k, v), g)
        with torch.no_grad():
            want = document(q.double(), k[first:].double(), v[first:].double(), None, None, None, g.double(), 1.0, dtype)
        what = "%s away, %s first" % (away, first)
        check(y.detach(), *want["y"], "y, " + what)
        check(gk[first:], *want["gk"], "gk, " + what)
        check(gv[first:], *want["gv"], "gv, " + what)
        # (a key of infinity meets zeros where a tile of queries is not full: still nothing)
        assert (gk[:first] == 0).all() and (gv[:first] == 0).all(), what


def far_points(gelib, dim, nq, nk, first, dtype, where, heads=4, kv=2):
    """The first keys lie `where` along a coordinate."""
    gen = torch.Generator(device="cuda").manual_seed(first + nq + dim)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)
    for away in AWAY:
        q, g = randn(nq, heads, dim).to(dtype), randn(nq, heads, dim).to(dtype)
        k, v = randn(first + nk, kv, dim).to(dtype), randn(first + nk, kv, dim).to(dtype)
        x, xk, slopes = randn(nq, 3), randn(first + nk, 3), torch.rand(heads, device="cuda", generator=gen) + 0.5
        xk[:, 0] += away
        xk[:first, 1] = where
        leaves = {"gq": q, "gk": k, "gv": v, "gx": x, "gslopes": slopes, "gxk": xk}
        for t in leaves.values():
            t.requires_grad_()
        marks = dict(starts=torch.tensor([0, first + nk], device="cuda", dtype=torch.int32), query_starts=torch.tensor([0, nq], device="cuda", dtype=torch.int32))
        y = gelib.attention(q, k, v, x, slopes, key_points=xk, **marks)
        got = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), g, retain_graph=True)), y=y.detach())
        plain = torch.autograd.grad(y, (q, k, v), g)   # (other kernels: without gradients of points)
        with torch.no_grad():
            want = document(q.double(), k[first:].double(), v[first:].double(), x.double(), xk[first:].double(), slopes.double(), g.double(), dim ** -0.5, dtype)
        for name, (value, tol) in want.items():
            t = got[name]
            if name in ("gk", "gv", "gxk"):
                assert (t[:first] == 0).all(), name
                t = t[first:]
            check(t, value, tol, "%s, %s away, %s first" % (name, away, first))
        for name, t in zip(("gq", "gk", "gv"), plain):
            value, tol = want[name]
            check(t if name == "gq" else t[first:], value, tol, "%s by itself, %s away, %s first" % (name, away, first))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("first", FIRST)
@pytest.mark.parametrize("nq,nk", OTHERS, ids=lambda v: str(v))
@pytest.mark.parametrize("dim", [16, 64, 128])
def test_finite_scores_without_a_share(gelib, dim, nq, nk, first, dtype):
    """Points 1e15 away: a maximum from there is off by more than all that the others differ by."""
    far_points(gelib, dim, nq, nk, first, dtype, 1e15)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("first", [3, 128, 1500])
@pytest.mark.parametrize("nq,nk", OTHERS, ids=lambda v: str(v))
@pytest.mark.parametrize("heads,kv", [(4, 2), (3, 3)])
def test_distances_whose_square_overflows(gelib, heads, kv, nq, nk, first, dtype):
    """Points 1e20 away and more are keys without a share, in gradients as in values; those of points in the neighbourhood are what they are without them."""
    for where in (1e20, -3e37):
        far_points(gelib, 32, nq, nk, first, dtype, where, heads, kv)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_a_head_without_slope_beside_far_points(gelib, dtype):
    """A slope of zero: the distance does not count, whatever it is."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    for nq, nk in ((5, 70), (130, 200)):
        q, k, v, g = (torch.randn(n, 2, 32, device="cuda", generator=gen).to(dtype) for n in (nq, nk, nk, nq))
        x, xk, slopes = torch.randn(nq, 3, device="cuda", generator=gen), torch.randn(nk, 3, device="cuda", generator=gen), torch.zeros(2, device="cuda")
        xk[::3, 2] = 1e30
        leaves = [t.requires_grad_() for t in (q, k, v, x, xk)]
        y = gelib.attention(q[None], k[None], v[None], x[None], slopes, key_points=xk[None])[0]
        got = dict(zip(("gq", "gk", "gv", "gx", "gxk"), torch.autograd.grad(y, leaves, g)), y=y.detach())
        with torch.no_grad():
            want = document(q.double(), k.double(), v.double(), None, None, None, g.double(), 32 ** -0.5, dtype)
        assert (got.pop("gx") == 0).all() and (got.pop("gxk") == 0).all()
        for name, t in got.items():
            check(t, *want[name], name)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("apart", [3e3, 1e5])
def test_maximum_grows_by_much(gelib, apart, dtype):
    """The first keys have weights until nearer ones come, a step at a time: no digit of the nearer ones' scores is lost."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    for nq, nk in ((3, 260), (100, 320)):
        q, k, v = (torch.randn(n, 2, 32, device="cuda", generator=gen).to(dtype) for n in (nq, nk, nk))
        x, xk, slopes = torch.randn(nq, 3, device="cuda", generator=gen), torch.randn(nk, 3, device="cuda", generator=gen), torch.ones(2, device="cuda")
        xk[:, 0] += apart * (4 - torch.arange(nk, device="cuda") // 64).clamp(min=0)
        last = nk - 256
        y = gelib.attention(q[None], k[None], v[None], x[None], slopes, key_points=xk[None])[0]
        want = document(q.double(), k[-last:].double(), v[-last:].double(), x.double(), xk[-last:].double(), slopes.double(), torch.zeros_like(q).double(), 32 ** -0.5, dtype)["y"]
        check(y, *want, "%s keys" % nk)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("points", [False, True], ids=["plain", "points"])
def test_scales(gelib, points, dtype):
    """Scales of zero (all keys alike, up to their distance), below it, and far from one.  A weight below 2^-126 may be zero (the hardware's
    exponential has no results between): besides, each is off by that, and the gradient of its score by that times gy . v - D."""
    gen = torch.Generator(device="cuda").manual_seed(11)
    for nq, nk in ((7, 90), (100, 333)):
        for scale in (0., -0., -1., 1e-20, -1e-30, 30.):
            q, k, v, g = (torch.randn(n, 2, 32, device="cuda", generator=gen).to(dtype) for n in (nq, nk, nk, nq))
            geo = [None] * 3
            if points:
                geo = [torch.randn(nq, 3, device="cuda", generator=gen), torch.randn(nk, 3, device="cuda", generator=gen), torch.rand(2, device="cuda", generator=gen)]
            leaves = [t.requires_grad_() for t in (q, k, v)]
            y = gelib.attention(q[None], k[None], v[None], geo[0] if geo[0] is None else geo[0][None], geo[2], key_points=geo[1] if geo[1] is None else geo[1][None], scale=scale,
                                lengths=torch.tensor([nk - 5], device="cuda", dtype=torch.int32))[0]
            got = dict(zip(("gq", "gk", "gv"), torch.autograd.grad(y, leaves, g)), y=y.detach())
            with torch.no_grad():
                d = [t if t is None else t.double() for t in geo]
                want = document(q.double(), k[:-5].double(), v[:-5].double(), d[0], d[1] if d[1] is None else d[1][:-5], d[2], g.double(), scale, dtype)
                kk, vv, qq, gg = (t.double().abs() for t in (k[:-5], v[:-5], q, g))
                dp = 2 * (gg.transpose(0, 1) @ vv.permute(1, 2, 0)).amax((1, 2))[:, None]
                few = {"y": vv.sum(0), "gv": gg.sum(0), "gq": abs(scale) * dp * kk.sum(0), "gk": abs(scale) * dp * qq.sum(0)}
            for name, t in got.items():
                check(t if name in ("y", "gq") else t[:-5], want[name][0], want[name][1] + 2.0 ** -126 * few[name], "%s, scale %s" % (name, scale))
