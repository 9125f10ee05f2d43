"""attention and linear_cross_entropy by torch's own operations (second derivatives, function transforms, forward mode): what does not exist is not
read there either.  It holds NaN here -- queries, keys, values, points, gradients and tangents of rows that are not there, rows that a loss leaves
out, weights that only those would meet -- and every derivative of what exists is that of the same call with zeros in those places,
to the bit: masked places are zero before anything is computed from them."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import torch.autograd.forward_ad as fwad  # noqa: E402

import gelib_amd as gelib  # noqa: E402

NAN = float("nan")


def cases(dtype):
    """(name, function of its real tensors, the tensors, for each of them a mask of what does not exist)"""
    gen = torch.Generator(device="cuda").manual_seed(5)

    def randn(*s):
        return torch.randn(*s, device="cuda", generator=gen).to(dtype)

    def index(*v):
        return torch.tensor(v, device="cuda", dtype=torch.int32)

    def points(*s):
        return torch.randn(*s, 3, device="cuda", generator=gen)

    def beyond(lengths, n):
        return torch.arange(n, device="cuda") >= lengths[:, None]
    slopes = torch.rand(4, device="cuda", generator=gen) + 0.5
    none = torch.zeros(4, dtype=torch.bool, device="cuda")
    n, m = index(6, 2, 0, 1), index(3, 0, 5, 7)
    gone, gone_k = beyond(n, 6), beyond(m, 7)
    out = [("padded, shared points", lambda q, k, v, p, s: gelib.attention(q, k, v, p, s, lengths=n, query_lengths=n),
            (randn(4, 6, 4, 8), randn(4, 6, 2, 8), randn(4, 6, 2, 8), points(4, 6), slopes), (gone, gone, gone, gone, none)),
           ("padded, two kinds of points", lambda q, k, v, p, s, pk: gelib.attention(q, k, v, p, s, key_points=pk, lengths=m, query_lengths=n),
            (randn(4, 6, 4, 8), randn(4, 7, 2, 8), randn(4, 7, 2, 8), points(4, 6), slopes, points(4, 7)), (gone, gone_k, gone_k, gone, none, gone_k)),
           ("padded, lengths of keys only", lambda q, k, v: gelib.attention(q, k, v, lengths=n), (randn(4, 5, 4, 8), randn(4, 6, 2, 8), randn(4, 6, 2, 8)),
            (torch.zeros(4, 5, dtype=torch.bool, device="cuda"), gone, gone))]
    starts, starts_k = index(2, 5, 5, 9), index(1, 4, 6, 6)
    row = torch.arange(11, device="cuda")
    gone, gone_k = (row < 2) | (row >= 9), (row[:8] < 1) | (row[:8] >= 6)
    out += [("packed, shared points", lambda q, k, v, p, s: gelib.attention(q, k, v, p, s, starts=starts),
             (randn(11, 4, 8), randn(11, 2, 8), randn(11, 2, 8), points(11), slopes), (gone, gone, gone, gone, none)),
            ("packed, two kinds of points", lambda q, k, v, p, s, pk: gelib.attention(q, k, v, p, s, key_points=pk, starts=starts_k, query_starts=starts),
             (randn(11, 4, 8), randn(8, 2, 8), randn(8, 2, 8), points(11), slopes, points(8)), (gone, gone_k, gone_k, gone, none, gone_k))]
    targets = torch.tensor([0, 5, -1, 2, -100, 1, 4, 3, -1], device="cuda")
    whole = torch.zeros(20, dtype=torch.bool, device="cuda")
    out.append(("loss", lambda x, w, b: gelib.linear_cross_entropy(x, w, targets, b), (randn(9, 20), randn(20, 6) / 4, randn(6)), (targets < 0, whole, whole[:6])))
    return out


def with_(value, ts, gone):
    return [t.masked_fill(g.view(*g.shape, *[1] * (t.dim() - g.dim())), value) for t, g in zip(ts, gone)]


TYPES = [torch.float32, torch.bfloat16]
CASES = range(6)


def same(got, want, name):
    for i, (a, b) in enumerate(zip(got, want)):
        assert torch.isfinite(b).all() and torch.equal(a, b), "%s: %s" % (name, i)


def weights(y, gone):
    gen = torch.Generator(device="cuda").manual_seed(2)
    g = torch.randn(y.shape, device="cuda", generator=gen).to(y.dtype)
    return g.masked_fill(gone.view(*gone.shape, *[1] * (g.dim() - gone.dim())), NAN)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("case", CASES)
def test_gradients_with_a_graph(case, dtype):
    name, f, ts, gone = cases(dtype)[case]
    results = []
    for value in (NAN, 0.):
        leaves = [t.requires_grad_() for t in with_(value, ts, gone)]
        y = f(*leaves)
        grads = torch.autograd.grad(y, leaves, weights(y, gone[0]), create_graph=True)
        again = torch.autograd.grad(sum((g.float() ** 2).sum() for g in grads), leaves)
        results.append([t.detach() for t in (y, *grads, *again)])
        # and the kernels' gradients of the same call
        for a, b in zip(grads, torch.autograd.grad(f(*leaves), leaves, weights(y, gone[0]))):
            assert torch.isfinite(b).all() and (a.float() - b.float()).abs().max() <= (1e-4 if dtype == torch.float32 else 0.03) * b.float().abs().max(), name
    same(*results, name)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("case", CASES)
def test_function_transforms(case, dtype):
    from torch.func import jvp, vjp, vmap
    name, f, ts, gone = cases(dtype)[case]
    results = []
    for value in (NAN, 0.):
        spoiled = with_(value, ts, gone)
        y, back = vjp(f, *spoiled)
        grads = back(weights(y, gone[0]))
        value_, tangent = jvp(f, tuple(spoiled), tuple(with_(value, [torch.ones_like(t) for t in ts], gone)))
        both = vmap(lambda t: f(t, *spoiled[1:]))(torch.stack([spoiled[0], 2 * spoiled[0]]))
        results.append([y, *grads, value_, tangent, both])
    same(*results, name)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("case", CASES)
def test_tangents(case, dtype):
    name, f, ts, gone = cases(dtype)[case]
    results = []
    for value in (NAN, 0.):
        with fwad.dual_level():
            duals = [fwad.make_dual(t, d) for t, d in zip(with_(value, ts, gone), with_(value, [torch.ones_like(t) for t in ts], gone))]
            results.append([t.clone() for t in fwad.unpack_dual(f(*duals))])
    same(*results, name)


def test_rows_left_out_and_infinite_weights():
    """A row that is left out meets nothing: not an infinite weight either, of a channel that all the other rows have zeros ... and -infinity of the class in."""
    targets = torch.tensor([2, -1, 0, -7], device="cuda")
    x = torch.randn(4, 5, device="cuda")
    x[:, 3] = torch.tensor([1., -2., 1., 0.], device="cuda")
    w = torch.randn(5, 4, device="cuda")
    w[3, 1] = float("-inf")   # (class 1 has no share in rows 0 and 2)
    leaves = [t.requires_grad_() for t in (x, w)]
    loss = gelib.linear_cross_entropy(x, w, targets)
    gx, gw = torch.autograd.grad(loss.sum(), leaves, create_graph=True)
    assert torch.isfinite(loss).all() and (gx[[1, 3]] == 0).all() and torch.isfinite(gw).all()
