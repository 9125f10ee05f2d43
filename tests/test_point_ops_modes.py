"""embedding, attention and linear_cross_entropy where only torch's own operations will do -- forward-mode derivatives, function transforms, tracing,
second derivatives -- are those operations: a derivative is never lost, a trace holds no memory that nobody has written.

Tolerances: derivatives of the two forms are compared in float32, which each of them rounds a few hundred times: 1e-4 of the largest."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

import gelib_amd as gelib

pytestmark = pytest.mark.gpu


def cases():
    """(function of its real tensors, the tensors)"""
    gen = torch.Generator(device="cuda").manual_seed(5)

    def randn(*s):
        return torch.randn(*s, device="cuda", generator=gen)

    def index(*v):
        return torch.tensor(v, device="cuda")
    tokens, targets = index(3, 0, 3, -1, 4, 1, 2), index(0, 5, -1, 2, 2, 1, 4, 3, 3)
    lengths, starts = index(6, 2, 1).int(), index(0, 4, 4, 9).int()
    return [
        (lambda table: gelib.embedding(tokens, table, 0.5), (randn(5, 12),)),
        (lambda q, k, v, p, s: gelib.attention(q, k, v, p, s, lengths=lengths, query_lengths=lengths),
         (randn(3, 6, 4, 8), randn(3, 6, 2, 8), randn(3, 6, 2, 8), randn(3, 6, 3), 0.5 + randn(4).abs())),
        (lambda q, k, v: gelib.attention(q, k, v, starts=starts), (randn(9, 4, 8), randn(9, 2, 8), randn(9, 2, 8))),
        (lambda x, w, b: gelib.linear_cross_entropy(x, w, targets, b), (randn(9, 20), randn(20, 6) / 4, randn(6))),
    ]


CASES = range(4)


def near(a, b):
    return (a - b).abs().max() <= 1e-4 * b.abs().max()


def reverse(f, ts, v=None):
    leaves = [t.clone().requires_grad_() for t in ts]
    y = f(*leaves)
    return y, torch.autograd.grad(y, leaves, torch.ones_like(y) if v is None else v, retain_graph=True)


@pytest.mark.parametrize("case", CASES)
def test_tangents(case):
    """A tangent against reverse mode, <v, J t> = <J^T v, t>."""
    f, ts = cases()[case]
    tangents = [torch.randn_like(t) for t in ts]
    plain = f(*ts)
    for requires in (False, True):
        with fwad.dual_level():
            value, tangent = fwad.unpack_dual(f(*[fwad.make_dual(t.clone().requires_grad_(requires), d) for t, d in zip(ts, tangents)]))
            assert tangent is not None and near(value, plain)
            v = torch.randn_like(plain)
            terms = torch.cat([(g.double() * d).flatten() for g, d in zip(reverse(f, ts, v)[1], tangents)])
            assert abs((v.double() * tangent).sum() - terms.sum()) <= 1e-4 * terms.abs().sum()


@pytest.mark.parametrize("case", CASES)
def test_second_derivatives(case):
    """<gradient of <J^T v, t>, t> against differences of <J^T v, t> along t: float32 differences of 1e-2, 2e-2 of the sum of the terms."""
    f, ts = cases()[case]
    if case == 0:
        return   # (linear)
    ts, tangents = list(ts), [torch.randn_like(t) for t in ts]
    v = torch.randn_like(f(*ts))

    def slope(at, graph=False):
        leaves = [t.clone().requires_grad_() for t in at]
        grads = torch.autograd.grad(f(*leaves), leaves, v, create_graph=graph)
        terms = torch.cat([(g.double() * d).flatten() for g, d in zip(grads, tangents)])
        return leaves, terms.sum()
    leaves, s = slope(ts, True)
    terms = torch.cat([(g.double() * d).flatten() for g, d in zip(torch.autograd.grad(s, leaves), tangents)])
    h = 1e-2
    up, down = (slope([t + k * h * d for t, d in zip(ts, tangents)])[1] for k in (1, -1))
    assert abs((up - down) / (2 * h) - terms.sum()) <= 2e-2 * terms.abs().sum()


@pytest.mark.parametrize("case", CASES)
def test_traces(case):
    f, ts = cases()[case]
    for leaves in (ts, [t.clone().requires_grad_() for t in ts]):
        traced = torch.jit.trace(f, tuple(leaves))
        for _ in range(3):
            junk = [torch.full((n,), 7.0, device="cuda") for n in (54, 252, 4096)]
            del junk
            new = [t + 0.1 * torch.randn_like(t) for t in ts]
            assert near(traced(*new), f(*new))


@pytest.mark.parametrize("case", CASES)
def test_function_transforms(case):
    from torch.func import grad, jvp, vjp, vmap
    f, ts = cases()[case]
    y, want = reverse(f, ts)
    value, tangent = jvp(f, tuple(ts), tuple(torch.ones_like(t) for t in ts))
    assert near(value, y) and abs(tangent.double().sum() - sum(g.double().sum() for g in want)) <= 1e-4 * sum(g.abs().sum() for g in want)
    for a, b in zip(grad(lambda *a: f(*a).sum(), argnums=tuple(range(len(ts))))(*ts), want):
        assert near(a, b)
    for a, b in zip(vjp(f, *ts)[1](torch.ones_like(y)), want):
        assert near(a, b)
    both = vmap(lambda t: f(t, *ts[1:]))(torch.stack([ts[0], 2 * ts[0]]))
    assert near(both[0], y) and near(both[1], f(2 * ts[0], *ts[1:]))


@pytest.mark.parametrize("case", CASES)
def test_batches_of_gradients(case):
    f, ts = cases()[case]
    leaves = [t.clone().requires_grad_() for t in ts]
    y = f(*leaves)
    vs = torch.randn(3, *y.shape, device="cuda")
    got = torch.autograd.grad(y, leaves, vs, is_grads_batched=True, retain_graph=True)
    for i in range(3):
        for a, b in zip(got, torch.autograd.grad(y, leaves, vs[i], retain_graph=True)):
            assert near(a[i], b)


@pytest.mark.parametrize("case", CASES)
def test_autocast(case):
    """Gradients with a graph, and calls that are left to torch's operations, keep the types of their tensors under autocast."""
    f, ts = cases()[case]
    y, want = reverse(f, ts)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        leaves = [t.clone().requires_grad_() for t in ts]
        z = f(*leaves)
        for a, b in zip(torch.autograd.grad(z, leaves, torch.ones_like(z), create_graph=True), want):
            assert a.dtype == torch.float32 and near(a, b)
        with fwad.dual_level():
            value, _ = fwad.unpack_dual(f(*[fwad.make_dual(t, t) for t in ts]))
            assert value.dtype == torch.float32 and near(value, y)
