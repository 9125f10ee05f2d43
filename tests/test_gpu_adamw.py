"""AdamW against the formulas in float64, its 8-bit moments code by code against a host form in integers (tests/adamw_codes.py).
Tolerances: m and v are two products and a sum, 4 half ulps of the terms' moduli; the step is m over a root, 8 half ulps more of it."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests import adamw_codes as A  # noqa: E402

u = 2.0 ** -24
LR, B1, B2, EPS, DECAY = 3e-3, 0.9, 0.99, 1e-8, 0.02


@pytest.fixture(scope="module")
def gelib():
    assert torch.cuda.is_available()
    import gelib_amd
    return gelib_amd


def real(t):
    return torch.view_as_real(t.detach()) if t.is_complex() else t.detach()


def make(sizes, dtype, seed, grads=True):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(n):
        t = torch.randn(*n, 2, device="cuda", generator=gen)
        return torch.view_as_complex(t) if dtype == torch.complex64 else t[..., 0].to(dtype).contiguous()
    params = [torch.nn.Parameter(randn(n)) for n in sizes]
    if grads:
        for p in params:
            p.grad = randn(p.shape)
    return params


# tensors of one element, around a block of 256, of several; more than a launch's table takes; an empty one
SIZES = [[(1,)], [(5, 51), (256,), (257,), (1, 3)], [(k % 7 + 1, 40) for k in range(150)], [(0,), (70000,)], [(3,), (0, 4), (1 << 20,), (999,)]]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.complex64], ids=str)
@pytest.mark.parametrize("sizes", SIZES, ids=[str(i) for i in range(len(SIZES))])
def test_32_bits(gelib, sizes, dtype):
    params = make(sizes, dtype, 1)
    opt = gelib.AdamW(params, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=DECAY)
    m, v = [torch.zeros_like(real(p), dtype=torch.float64) for p in params], [torch.zeros_like(real(p), dtype=torch.float64) for p in params]
    for t in range(1, 4):
        before = [real(p).double() for p in params]
        opt.step()
        for k, p in enumerate(params):
            g = real(p.grad).double()
            m[k] = B1 * m[k] + (1 - B1) * g
            v[k] = B2 * v[k] + (1 - B2) * g * g
            tol_m, tol_v = 4 * t * u * (m[k].abs() + g.abs()), 4 * t * u * (v[k] + g * g)
            gm, gv = opt.moments(p)
            assert gm.shape == real(p).shape
            assert ((gm.double() - m[k]).abs() <= tol_m).all() and ((gv.double() - v[k]).abs() <= tol_v).all()
            step = LR / (1 - B1 ** t) * m[k] / ((v[k] / (1 - B2 ** t)).sqrt() + EPS)
            want = before[k] * (1 - LR * DECAY) - step
            dstep = LR / (1 - B1 ** t) * tol_m / ((v[k] / (1 - B2 ** t)).sqrt() + EPS) + step.abs() * (8 * u + 8 * t * u)
            tol = dstep + 2 * u * (before[k].abs() + step.abs())
            if dtype == torch.bfloat16:   # rounded up or down: a whole unit, 2^-7 of the value
                tol = tol + 2.0 ** -7 * want.abs()
            assert ((real(p).double() - want).abs() <= tol).all(), (k, t)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.complex64], ids=str)
@pytest.mark.parametrize("sizes", SIZES, ids=[str(i) for i in range(len(SIZES))])
def test_8_bits_code_by_code(gelib, sizes, dtype):
    params = make(sizes, dtype, 2)
    opt = gelib.AdamW(params, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=DECAY, state_bits=8, seed=12345678901)
    m, v = ([np.zeros(real(p).numel(), np.float32) for p in params] for _ in range(2))
    for t in range(1, 4):
        before = [real(p).float().cpu().numpy().ravel() for p in params]
        opt.step()
        for k, p in enumerate(params):
            g = real(p.grad).float().cpu().numpy().ravel()
            first = opt._places[p][0]
            nm, nv, np_ = A.step(before[k], g, m[k], v[k], LR, B1, B2, EPS, DECAY, t)
            h, h2 = A.random_bits(first + np.arange(len(g)), t, 12345678901)
            m[k], v[k] = A.kept(nm, h & 0xfffff, 126, False), A.kept(nv, h >> 12, 254, True)
            gm, gv = opt.moments(p)
            assert gm.dtype == torch.bfloat16
            assert np.array_equal(gm.float().cpu().numpy().ravel(), m[k]) and np.array_equal(gv.float().cpu().numpy().ravel(), v[k]), (k, t)
            got = real(p).float().cpu().numpy().ravel()
            if dtype == torch.bfloat16:
                assert np.array_equal(got, A.to_bfloat16(np_, h2))
            else:
                assert (np.abs(got - np_) <= 4 * u * (np.abs(before[k]) + np.abs(np_))).all()
    am, av = opt.moments()
    opt.set_moments(am, av, 3)   # what it told comes back as it was
    for a, b in zip(opt.moments(), (am, av)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_places_in_memory(gelib, bits, dtype):
    """Parameters and gradients at any multiple of their element, between elements that nobody writes."""
    outs = []
    for shift in (0, 1, 3):
        gen = torch.Generator(device="cuda").manual_seed(9)
        buf, params = torch.full((6000,), 7.0, device="cuda", dtype=dtype), []
        at = 0
        for n in (1, 255, 256, 700, 1030):
            p = torch.nn.Parameter(buf[at + shift:at + shift + n])
            p.data.copy_(torch.randn(n, device="cuda", generator=gen))
            p.grad = torch.empty(n + 3, device="cuda", dtype=dtype)[shift:shift + n].copy_(torch.randn(n, device="cuda", generator=gen))
            params.append(p)
            at += n + 8
        opt = gelib.AdamW(params, state_bits=bits)
        opt.step()
        opt.step()
        outs.append([p.detach().clone() for p in params] + list(opt.moments()))
        with torch.no_grad():
            for p in params:
                p.fill_(7.0)
        assert (buf == 7.0).all()
    for other in outs[1:]:
        for a, b in zip(outs[0], other):
            assert torch.equal(a, b)


@pytest.mark.parametrize("bits", [8, 32])
def test_groups_missing_gradients_and_state(gelib, bits):
    params = make([(300,), (20, 30), (7,)], torch.float32, 4)
    copies = [torch.nn.Parameter(p.detach().clone()) for p in params]
    for c, p in zip(copies, params):
        c.grad = p.grad.clone()

    def build(ps):
        return gelib.AdamW([{"params": ps[:1]}, {"params": ps[1:], "lr": 0.1, "weight_decay": 0.0}], lr=1e-2, state_bits=bits, seed=5)
    a, b = build(params), build(copies)
    params[1].grad, kept = None, params[1].grad
    was = params[1].detach().clone()
    a.step()
    assert torch.equal(params[1], was) and not a.moments(params[1])[0].any() and [list(g.steps) for g in a._groups] == [[1], [0, 1]]
    params[1].grad = kept
    copies[1].grad, kept = None, copies[1].grad
    b.step()
    copies[1].grad = kept
    saved = a.state_dict()
    a.step()
    b.load_state_dict(saved)
    b.step()
    for p, q in zip(params, copies):
        assert torch.equal(p, q)
    for p, q in zip(a.moments(), b.moments()):
        assert torch.equal(p, q)
    # the first step of a parameter moves by lr, whenever it comes
    moved = (params[1].detach() - was).abs()
    assert ((moved - 0.1).abs() < 1e-5).all()


def test_a_group_that_comes_later(gelib):
    a, b = make([(300,)], torch.float32, 4), make([(77,)], torch.float32, 5)
    opt = gelib.AdamW(a, state_bits=8)
    opt.step()
    kept = [t.clone() for t in opt.moments(a[0])]
    opt.add_param_group({"params": b, "lr": 0.5, "weight_decay": 0.0})
    for x, y in zip(opt.moments(a[0]), kept):
        assert torch.equal(x, y)
    was = b[0].detach().clone()
    opt.step()
    assert ((b[0].detach() - was).abs() - 0.5).abs().max() < 1e-5 and [list(g.steps) for g in opt._groups] == [[2], [1]]
    b[0].data = torch.zeros(5000, device="cuda")   # no room for its moments
    b[0].grad = torch.zeros(5000, device="cuda")
    with pytest.raises(ValueError):
        opt.step()


def test_scheduler_closure_zero_grad(gelib):
    p = torch.nn.Parameter(torch.ones(10, device="cuda"))
    opt = gelib.AdamW([p], lr=0.5, weight_decay=0.0)
    scheduler = torch.optim.lr_scheduler.StepLR(opt, 1, 0.1)

    def closure():
        opt.zero_grad()
        loss = p.sum()
        loss.backward()
        return loss
    assert float(opt.step(closure)) == 10.0
    scheduler.step()
    opt.step(closure)
    assert torch.allclose(p, torch.full_like(p, 1 - 0.5 - 0.05))


def test_not_finite_and_zero(gelib):
    for bits in (8, 32):
        p = torch.nn.Parameter(torch.ones(600, device="cuda"))
        p.grad = torch.full((600,), 1e-3, device="cuda")
        p.grad[5], p.grad[6], p.grad[7], p.grad[300:] = float("nan"), float("inf"), 1e30, 0.0
        opt = gelib.AdamW([p], lr=1e-2, weight_decay=0.0, state_bits=bits)
        for _ in range(3):
            opt.step()
        bad = torch.zeros(600, dtype=torch.bool, device="cuda")
        bad[5:7] = True
        assert torch.equal(torch.isnan(p), bad)
        assert p[7] == 1   # its square is infinite
        # the neighbours in the block keep their scale: three steps of lr (8 bits: m is known to a sixteenth, v to an eighth)
        assert (((1 - p[~bad][:200] - 0.03).abs() < (1e-5 if bits == 32 else 4e-3)) | (p[~bad][:200] == 1)).all() and (p[300:] == 1).all()
        assert (p[8:200] < 1).all()


def test_8_bits_follow_the_gradients(gelib):
    """A constant gradient g brings m to g and v to g^2: rounding at random is right on the average (65536 elements: the mean of v is within
    1 %), where rounding to the nearest would leave v below a tenth of it."""
    p = torch.nn.Parameter(torch.zeros(65536, device="cuda"))
    p.grad = torch.full_like(p, 0.3)
    opt = gelib.AdamW([p], lr=0.0, betas=(0.9, 0.99), state_bits=8)
    for _ in range(600):
        opt.step()
    m, v = (t.float() for t in opt.moments())
    assert abs(m.mean() / 0.3 - 1) < 0.01 and abs(v.mean() / 0.09 - 1) < 0.01


def test_bfloat16_parameters_move_by_small_steps(gelib):
    """Steps of a hundredth of a unit in the last place: 1000 of them are 10 units on the average."""
    p = torch.nn.Parameter(torch.full((65536,), 1.5, device="cuda", dtype=torch.bfloat16))
    p.grad = torch.ones_like(p)
    opt = gelib.AdamW([p], lr=2.0 ** -7 / 100, weight_decay=0.0)
    for _ in range(1000):
        opt.step()
    moved = (1.5 - p.float()).mean() / 2.0 ** -7
    assert abs(float(moved) - 10) < 0.1


def test_large_arrays(gelib):
    """Places beyond 2^31 elements (bfloat16 parameters, 8-bit moments: 13 GB)."""
    n = (1 << 31) + 5000
    p = torch.nn.Parameter(torch.zeros(n, device="cuda", dtype=torch.bfloat16))
    q = torch.nn.Parameter(torch.zeros(300, device="cuda"))
    p.grad, q.grad = torch.zeros_like(p), torch.ones_like(q)
    p.grad[-3:] = 1
    opt = gelib.AdamW([p, q], lr=1.0, weight_decay=0.0, state_bits=8)
    opt.step()
    torch.cuda.synchronize()
    assert (p[-3:] == -1).all() and not p[:-3].any() and (q == -1).all()
    m, v = opt.moments(q)
    assert ((m.float() - 0.1).abs() < 0.02).all() and ((v.float() - 1e-3).abs() < 2e-4).all()


def test_another_stream(gelib):
    outs = []
    for side in (torch.cuda.current_stream(), torch.cuda.Stream()):
        params = make([(3000,), (40, 40)], torch.float32, 6)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            opt = gelib.AdamW(params, state_bits=8)
            opt.step()
            opt.step()
        torch.cuda.current_stream().wait_stream(side)
        outs.append([p.detach().clone() for p in params])
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_refusals(gelib):
    p = make([(30,)], torch.float32, 1)
    for bad, error in ((lambda: gelib.AdamW(p, state_bits=16), ValueError), (lambda: gelib.AdamW(p, lr=-1.0), ValueError),
                       (lambda: gelib.AdamW(p, betas=(1.0, 0.9)), ValueError), (lambda: gelib.AdamW(make([(3,)], torch.float16, 1)), TypeError),
                       (lambda: gelib.AdamW([torch.nn.Parameter(torch.zeros(3))]), ValueError),
                       (lambda: gelib.AdamW([torch.nn.Parameter(torch.zeros(4, 3, device="cuda").t())]), ValueError),
                       (lambda: gelib.AdamW(p).set_moments(torch.zeros(3), torch.zeros(3), 1), ValueError)):
        with pytest.raises(error):
            bad()
    opt = gelib.AdamW(p)
    with pytest.raises(ValueError):
        gelib.AdamW(p, state_bits=8).load_state_dict(opt.state_dict())
    assert math.isfinite(float(p[0].sum()))
