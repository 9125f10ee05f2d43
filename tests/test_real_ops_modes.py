"""group_norm_act and linear_act where only torch's own operations will do -- forward-mode derivatives, function transforms, tracing,
dispatch modes -- are those operations: a derivative is never lost, a trace holds no memory that nobody has written.

Tolerances: derivatives of the two forms are compared in float32, which each of them rounds a few hundred times: 1e-4 of the largest."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

import gelib_amd as gelib


def linear(x, w, b, r):
    return gelib.linear_act(x, w, b, residual=r, act="silu")


def norm(x, w, b, lengths):
    return gelib.group_norm_act(x, 3, w, b, act="gelu", lengths=lengths)


def cases():
    gen = torch.Generator(device="cuda").manual_seed(3)

    def randn(*s):
        return torch.randn(*s, device="cuda", generator=gen)
    lengths = torch.tensor([7, 3, 0], device="cuda", dtype=torch.int32)
    return [(linear, (randn(9, 20), randn(20, 6) / 4, randn(6), randn(9, 6)), 4), (norm, (randn(3, 7, 12), 1 + 0.1 * randn(12), randn(12), lengths), 3)]


def near(a, b):
    return (a - b).abs().max() <= 1e-4 * b.abs().max()


def test_shapes_without_data():
    """(Runs without a GPU.)"""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x, w = (torch.empty(*s, device="cuda", dtype=torch.bfloat16) for s in ((4, 5, 8), (8, 6)))
        lengths = torch.empty(4, device="cuda", dtype=torch.int32)
        for y, last in ((gelib.linear_act(x, w, act="gelu"), 6), (gelib.group_norm_act(x, 2, act="silu", lengths=lengths), 8)):
            assert y.shape == (4, 5, last) and y.dtype == torch.bfloat16 and y.is_cuda
        with pytest.raises(ValueError):
            gelib.linear_act(x, w, residual=x)
        with pytest.raises(ValueError):
            gelib.group_norm_act(x, 3)
        with pytest.raises(ValueError):
            gelib.group_norm_act(x, 2, eps=-1.0)
        with pytest.raises(ValueError):
            gelib.linear_act(x, w, act="tanh")


@pytest.mark.gpu
def test_tangents():
    """A tangent against reverse mode, <v, J t> = <J^T v, t>, and against differences (2e-3 of the sum: third derivatives, rounding)."""
    for f, ts, k in cases():
        gen = torch.Generator(device="cuda").manual_seed(4)
        tangents = [torch.randn(t.shape, device="cuda", generator=gen) for t in ts[:k]]
        for requires in (False, True):
            leaves = [t.clone().requires_grad_(requires) for t in ts[:k]]
            with fwad.dual_level():
                y = f(*[fwad.make_dual(t, d) for t, d in zip(leaves, tangents)], *ts[k:])
                value, tangent = fwad.unpack_dual(y)
                assert tangent is not None
                value, tangent = value.detach().clone(), tangent.detach().clone()
            plain = f(*ts)
            assert near(value, plain)
            v = torch.randn(plain.shape, device="cuda", generator=gen)
            leaves = [t.clone().requires_grad_() for t in ts[:k]]
            grads = torch.autograd.grad(f(*leaves, *ts[k:]), leaves, v)
            terms = torch.cat([(g.double() * d).flatten() for g, d in zip(grads, tangents)])
            assert abs((v.double() * tangent).sum() - terms.sum()) <= 1e-4 * terms.abs().sum()
            h = 1e-2
            up, down = (f(*[t + s * h * d for t, d in zip(ts, tangents)], *ts[k:]).double() for s in (1, -1))
            assert abs(((up - down) / (2 * h) * v).sum() - terms.sum()) <= 2e-3 * terms.abs().sum()


@pytest.mark.gpu
def test_tangents_of_a_gradient():
    """The gradient that comes in has a tangent, the result was formed outside: the backward pass is linear in it."""
    for f, ts, k in cases():
        leaves = [t.clone().requires_grad_() for t in ts[:k]]
        y = f(*leaves, *ts[k:])
        g, d = torch.randn_like(y), torch.randn_like(y)
        want = torch.autograd.grad(y, leaves, d, retain_graph=True)
        values = torch.autograd.grad(y, leaves, g, retain_graph=True)
        with fwad.dual_level():
            for got, value, t in zip(torch.autograd.grad(y, leaves, fwad.make_dual(g, d)), values, want):
                got, tangent = fwad.unpack_dual(got)
                assert tangent is not None and near(tangent, t) and near(got, value) and not got.requires_grad


@pytest.mark.gpu
def test_traces():
    """A traced call computes: it gives what the kernels give, for other inputs and after memory has been written over."""
    for f, ts, k in cases():
        for leaves in (ts, [t.clone().requires_grad_(t.is_floating_point()) for t in ts]):
            traced = torch.jit.trace(f, tuple(leaves))
            for _ in range(3):
                junk = [torch.full((n,), 7.0, device="cuda") for n in (54, 252, 4096)]
                del junk
                new = [t + 0.1 * torch.randn_like(t) if t.is_floating_point() else t for t in ts]
                assert near(traced(*new), f(*new))


@pytest.mark.gpu
def test_function_transforms():
    from torch.func import grad, jvp, vjp, vmap
    for f, ts, k in cases():
        tangents = [torch.ones_like(t) for t in ts[:k]]
        value, tangent = jvp(lambda *a: f(*a, *ts[k:]), tuple(ts[:k]), tuple(tangents))
        leaves = [t.clone().requires_grad_() for t in ts[:k]]
        y = f(*leaves, *ts[k:])
        want = torch.autograd.grad(y, leaves, torch.ones_like(y), retain_graph=True)
        assert near(value, y) and abs((tangent.double().sum() - sum(g.double().sum() for g in want))) <= 1e-4 * sum(g.abs().sum() for g in want)
        got = grad(lambda *a: f(*a, *ts[k:]).sum(), argnums=tuple(range(k)))(*ts[:k])
        for a, b in zip(got, want):
            assert near(a, b)
        _, back = vjp(lambda *a: f(*a, *ts[k:]), *ts[:k])
        for a, b in zip(back(torch.ones_like(y)), want):
            assert near(a, b)
        many = torch.stack([ts[0], 2 * ts[0]])
        both = vmap(lambda x: f(x, *ts[1:]))(many)
        assert near(both[0], y) and near(both[1], f(2 * ts[0], *ts[1:]))


@pytest.mark.gpu
def test_autocast():
    """Gradients with a graph, and calls that are left to torch's operations, keep the types of their tensors under autocast."""
    for f, ts, k in cases():
        leaves = [t.clone().requires_grad_() for t in ts[:k]]
        y = f(*leaves, *ts[k:])
        v = torch.randn_like(y)
        want = torch.autograd.grad(y, leaves, v, retain_graph=True)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            for a, b in zip(torch.autograd.grad(f(*leaves, *ts[k:]), leaves, v, create_graph=True), want):
                assert a.dtype == torch.float32 and near(a, b)
            with fwad.dual_level():
                value, _ = fwad.unpack_dual(f(*[fwad.make_dual(t, t) for t in ts[:k]], *ts[k:]))
                assert value.dtype == torch.float32 and near(value, y)


@pytest.mark.gpu
def test_kernels_run_elsewhere():
    """After all of it, and beside it for tensors without a tangent, calls go to the kernels (path 7)."""
    from gelib_amd import cabi
    L = cabi.lib()
    for f, ts, k in cases():
        torch.func.vmap(lambda x: f(x, *ts[1:]))(torch.stack([ts[0], ts[0]]))
        for forward in (False, True):
            cabi.check(L.gelib_hip_adamw_step(0, None, None, None, None, None, None, None, None, None, 0, 32, 0.0, 0.0, 0.0, 0.0, 0.0, 0, None))
            assert L.gelib_hip_last_path() == 0
            if forward:
                with fwad.dual_level():
                    f(*ts)
            else:
                f(*ts)
            assert L.gelib_hip_last_path() == 7


@pytest.mark.gpu
def test_batches_of_gradients():
    """Several gradients of one result in one call, as a vectorised Jacobian asks for them."""
    for f, ts, k in cases():
        leaves = [t.clone().requires_grad_() for t in ts[:k]]
        y = f(*leaves, *ts[k:])
        vs = torch.randn(3, *y.shape, device="cuda")
        got = torch.autograd.grad(y, leaves, vs, is_grads_batched=True, retain_graph=True)
        for i in range(3):
            for a, b in zip(got, torch.autograd.grad(y, leaves, vs[i], retain_graph=True)):
                assert near(a[i], b)
