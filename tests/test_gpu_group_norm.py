"""group_norm_act and its gradients against the formulas in float64.  Tolerances, u = 2^-24: a sum of k terms formed in pieces is off by
(64 + k / 64) u of the sum of their moduli at most (chains of up to 64 terms and as many pieces); what is off in x - mean, rstd and z is
carried through the formulas; act' changes by 1.2 of a change of z (gelu, the steepest), for relu by 1 where z is within its error of
zero; results are rounded to their type once."""
import pytest

from tests import gpu_util as U  # noqa: F401

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

HALF_ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEAST = {torch.float32: 1e-44, torch.bfloat16: 1e-38, torch.float16: 2.0 ** -24}
u = 2.0 ** -24


@pytest.fixture(scope="module")
def gelib():
    assert torch.cuda.is_available()
    import gelib_amd
    return gelib_amd


def act64(z, act):
    F = torch.nn.functional
    return {"none": lambda t: t, "relu": F.relu, "silu": F.silu, "gelu": F.gelu}[act](z)


def slope64(z, act):
    if act == "relu":
        return (z > 0).double()
    z = z.detach().requires_grad_()
    with torch.enable_grad():
        return torch.autograd.grad(act64(z, act).sum(), z)[0] if act != "none" else torch.ones_like(z)


def check(got, want, tol, what):
    err = (got.double() - want).abs()
    tol = tol + HALF_ULP[got.dtype] * want.abs() + LEAST[got.dtype]
    assert torch.isfinite(got.double()).all(), what
    assert (err <= tol).all(), "%s: worst error / tolerance %.2f" % (what, (err / tol).max())


def reference(x, groups, w, b, eps, act, lengths, g=None):
    """{name: (value, tolerance)}; x (n, s, c) float64, lengths always given"""
    n, s, c = x.shape
    k = c // groups
    live = (torch.arange(s, device=x.device) < lengths[:, None])[:, :, None, None]
    t = torch.where(live, x.view(n, s, groups, k), 0.)
    cnt = (lengths.clamp(min=1) * k).double()[:, None, None, None]
    W, B = w.view(groups, k), b.view(groups, k)
    mean = t.sum((1, 3), keepdim=True) / cnt
    d = torch.where(live, t - mean, 0.)
    rstd = (d.square().sum((1, 3), keepdim=True) / cnt + eps).rsqrt()
    xh = d * rstd
    z = xh * W + B
    chain = (64 + cnt / 64) * u
    biggest = t.abs().amax((1, 3), keepdim=True)
    dxh = rstd * chain * biggest + 2 * chain * xh.abs()
    dz = dxh * W.abs() + 4 * u * (z.abs() + B.abs())
    out = {"y": (torch.where(live, act64(z, act), 0.), 1.2 * dz + 16 * u * z.abs() * (1 + z.abs()))}
    if g is not None:
        G = torch.where(live, g.view(n, s, groups, k), 0.)
        gz = G * slope64(z, act)
        dgz = G.abs() * (torch.where(z.abs() <= dz, 1., 0.) if act == "relu" else (0. if act == "none" else 1.2) * dz + 16 * u * (1 + z.abs()))
        q, dq = gz * W, dgz * W.abs() + 2 * u * (gz * W).abs()

        def mean_of(v, dv):
            return v.sum((1, 3), keepdim=True) / cnt, (dv + chain * v.abs()).sum((1, 3), keepdim=True) / cnt
        m1, dm1 = mean_of(q, dq)
        m2, dm2 = mean_of(q * xh, dq * xh.abs() + q.abs() * dxh)
        gx = torch.where(live, rstd * (q - m1 - xh * m2), 0.)
        dgx = rstd * (dq + dm1 + dxh * m2.abs() + xh.abs() * dm2 + 4 * u * (q.abs() + m1.abs() + (xh * m2).abs())) + 2 * chain * gx.abs()
        out["gx"] = gx, dgx
        terms = (64 + n * s / 64) * u
        out["gw"] = (gz * xh).sum((0, 1)), (dgz * xh.abs() + gz.abs() * dxh + terms * (gz * xh).abs()).sum((0, 1))
        out["gb"] = gz.sum((0, 1)), (dgz + terms * gz.abs()).sum((0, 1))
    return out


# samples, positions, channels, groups: single positions and values, odd everything, a group as wide as the sample, groups of one channel,
# vectors that straddle groups (3 and 10 channels), many small samples, long ones that are cut into pieces, wide rows
SHAPES = [(1, 1, 1, 1), (3, 1, 8, 2), (2, 5, 7, 7), (2, 19, 30, 10), (5, 33, 64, 8), (1, 130, 320, 32), (700, 1, 64, 8), (1300, 3, 24, 4), (1, 4097, 48, 3),
          (3, 2050, 96, 32), (2, 700, 1024, 1), (2, 9, 2056, 257), (1, 30011, 5, 1), (260, 70, 33, 11), (1, 3, 8200, 4)]


# groups wider than a block: in pieces, in as many pieces as channels (a prime number of them), one group of everything
SHAPES += [(2, 40, 4104, 1), (2, 5, 4106, 2), (300, 1, 9000, 3), (1, 700, 6144, 2), (2, 40, 2053, 1), (3, 400, 257, 1)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_values_and_gradients(gelib, shape, act, dtype):
    n, s, c, groups = shape
    gen = torch.Generator(device="cuda").manual_seed(n * 7 + s * 3 + c)

    def randn(*size):
        return torch.randn(*size, device="cuda", generator=gen)
    x = (randn(n, s, c) * (0.5 + randn(c).abs()) + 2 * randn(c)).to(dtype).requires_grad_()
    w, b = (1 + 0.3 * randn(c)).to(dtype).requires_grad_(), (0.5 * randn(c)).to(dtype).requires_grad_()
    g = randn(n, s, c).to(dtype)
    for ragged in (False, True) if s > 1 else (False,):
        lengths = torch.randint(0, s + 1, (n,), device="cuda", generator=gen, dtype=torch.int32) if ragged else None
        if ragged:
            lengths[0], lengths[-1] = 1, 0
        y = gelib.group_norm_act(x, groups, w, b, eps=1e-3, act=act, lengths=lengths)
        got = dict(zip(("gx", "gw", "gb"), torch.autograd.grad(y, (x, w, b), g)), y=y.detach())
        full = torch.full((n,), s, device="cuda") if lengths is None else lengths.long()
        with torch.no_grad():
            want = reference(x.double(), groups, w.double(), b.double(), 1e-3, act, full, g.double())
        for k in ("y", "gx", "gw", "gb"):
            v, tol = want[k]
            check(got[k], v.reshape(got[k].shape), tol.reshape(got[k].shape), "%s of %s, ragged %s" % (k, shape, ragged))
        if ragged:
            behind = torch.arange(s, device="cuda") >= lengths[:, None]
            assert not y[behind].any() and not got["gx"][behind].any()
        assert torch.equal(y, gelib.group_norm_act(x.detach(), groups, w.detach(), b.detach(), eps=1e-3, act=act, lengths=lengths))
        again = torch.autograd.grad(gelib.group_norm_act(x, groups, w, b, eps=1e-3, act=act, lengths=lengths), (x, w, b), g)
        for a, k in zip(again, ("gx", "gw", "gb")):
            assert torch.equal(a, got[k])   # fixed orders of summation


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_layouts(gelib, dtype):
    gen = torch.Generator(device="cuda").manual_seed(5)
    big = torch.randn(6, 9, 11, 80, device="cuda", generator=gen).to(dtype)
    views = [big[:, :, :, 5:37], big[1:5], big[:, 2:7, :, 8:24], big.transpose(1, 2), big[::2, :, :, :48], big[:, :, 3:4, :], big[:, :, :, ::2],
             big[:1, :1, :1, :8].expand(3, 5, 4, 8), big[..., 1:49].transpose(0, 1), torch.randn(4, 6, 7, device="cuda", dtype=dtype).permute(1, 2, 0)]
    for v in views:
        c = v.shape[-1]
        groups = 4 if c % 4 == 0 else 1
        p = v.contiguous().requires_grad_()
        q = v.detach().requires_grad_()
        a, b = (gelib.group_norm_act(t, groups, act="silu") for t in (p, q))
        g = torch.randn(v.shape, device="cuda", generator=gen).to(dtype)
        wide = torch.empty(*v.shape[:-1], c + 3, device="cuda", dtype=dtype)[..., 3:].copy_(g)   # rows that are not aligned
        assert torch.equal(a, b) and a.shape == v.shape and b.is_contiguous()
        want, = torch.autograd.grad(a, p, g)
        assert torch.equal(torch.autograd.grad(b, q, wide)[0], want)
        # a gradient that is broadcast
        a, b = (gelib.group_norm_act(t, groups, act="silu") for t in (p, q))
        assert torch.equal(torch.autograd.grad(a.sum(), p)[0], torch.autograd.grad(b.sum(), q)[0])


def test_values_behind_a_length_are_not_read(gelib):
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(5, 40, 32, device="cuda", generator=gen)
    g = torch.randn(5, 40, 32, device="cuda", generator=gen)
    lengths = torch.tensor([40, 0, 1, 17, -3], device="cuda", dtype=torch.int32)
    behind = torch.arange(40, device="cuda") >= lengths[:, None]

    def both(x, g):
        x = x.clone().requires_grad_()
        w = torch.ones(32, device="cuda", requires_grad=True)
        y = gelib.group_norm_act(x, 4, w, act="silu", lengths=lengths)
        return (y.detach(), *torch.autograd.grad(y, (x, w), g))
    want = both(x, g)
    for bad in (float("nan"), float("inf"), -3.4e38):
        px, pg = x.clone(), g.clone()
        px[behind], pg[behind] = bad, bad
        for a, b in zip(both(px, pg), want):
            assert torch.equal(a, b)
    # longer than the sample is the sample
    assert torch.equal(gelib.group_norm_act(x, 4, lengths=torch.full((5,), 1 << 30, device="cuda", dtype=torch.int32)), gelib.group_norm_act(x, 4))


@pytest.mark.parametrize("shape", [(70000, 3, 10304), (3, 2250000, 320)], ids=str)
def test_offsets_beyond_32_bits(gelib, shape):
    """4.3 GB tensors: the last sample is what it is by itself (the same kernels on the same values), and so is its gradient."""
    n, s, c = shape
    x = torch.zeros(shape, device="cuda", dtype=torch.bfloat16)
    x[-1].normal_()
    g = torch.zeros_like(x)
    g[-1].normal_()
    leaf, alone = x.requires_grad_(), x[-1:].detach().clone().requires_grad_()
    a, b = (gelib.group_norm_act(t, 32, act="silu") for t in (leaf, alone))
    assert torch.isfinite(a[0].float()).all()
    # (how a sample is cut may depend on how many there are: the order of sums, not more)
    assert (a[-1].float() - b[0].float()).abs().max() < 0.04
    ga, = torch.autograd.grad(a, leaf, g)
    gb, = torch.autograd.grad(b, alone, g[-1:])
    assert (ga[-1].float() - gb[0].float()).abs().max() < 0.04 and not ga[0].any()


def test_memory_beside_the_operands_is_not_touched_or_read(gelib):
    """Operands between NaNs and results between sentinels, through the C ABI, over every way that a call is cut."""
    from gelib_amd import cabi
    L = cabi.lib()
    for dtype, code in ((torch.float32, 0), (torch.bfloat16, 1)):
        for n, s, c, groups in ((3, 5, 12, 3), (2, 33, 30, 10), (700, 1, 64, 8), (1, 2500, 48, 6), (2, 300, 7, 1), (1, 4, 8200, 4)):
            def framed(shape, fill=None, frame=float("nan"), t=dtype):
                size = 1
                for k in shape:
                    size *= k
                whole = torch.full((size + 1024,), frame, device="cuda", dtype=t)
                inner = whole[512:512 + size].view(shape)
                inner.normal_() if fill is None else inner.fill_(fill)
                return whole, inner
            (X, x), (W, w), (B, b), (G, g) = framed((n, s, c)), framed((c,)), framed((c,)), framed((n, s, c))
            outs = [framed(k, 3.0, 5.0) for k in ((n, s, c), (n, s, c), (c,), (c,))]
            (M, mean), (R, rstd) = (framed((n, groups), 3.0, 5.0, torch.float32) for _ in range(2))
            y, gx, gw, gb = (t for _, t in outs)
            stream = torch.cuda.current_stream().cuda_stream
            P = [t.data_ptr() for t in (x, w, b, g)]

            def work(back):
                need = L.gelib_hip_group_norm_act_workspace_bytes(back, code, n, s, c, groups)
                return torch.full((max(need, 16),), 255, device="cuda", dtype=torch.uint8), need
            ws, need = work(0)
            cabi.check(L.gelib_hip_group_norm_act_fwd(y.data_ptr(), mean.data_ptr(), rstd.data_ptr(), P[0], P[1], P[2], None, code, n, s, c, groups, s * c, c, 1e-3, 2,
                                                      ws.data_ptr(), need, stream))
            ws, need = work(1)
            cabi.check(L.gelib_hip_group_norm_act_bwd(gx.data_ptr(), gw.data_ptr(), gb.data_ptr(), P[3], mean.data_ptr(), rstd.data_ptr(), P[0], P[1], P[2], None, code,
                                                      n, s, c, groups, s * c, c, 2, ws.data_ptr(), need, stream))
            with torch.no_grad():
                want = reference(x.double(), groups, w.double(), b.double(), 1e-3, "silu", torch.full((n,), s, device="cuda"), g.double())
            for got, k in ((y, "y"), (gx, "gx"), (gw, "gw"), (gb, "gb")):
                v, tol = want[k]
                check(got, v.reshape(got.shape), tol.reshape(got.shape), "%s of %s" % (k, (n, s, c, groups)))
            for t in [t for t, _ in outs] + [M, R]:
                assert (t[:512] == 5).all() and (t[-512:] == 5).all()


def test_large_mean(gelib):
    """Statistics are formed around the mean: a thousand standard deviations of it cost three digits, not six."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    for shape in ((2, 60, 64, 4), (1, 20000, 64, 4)):
        n, s, c, groups = shape
        x = torch.randn(n, s, c, device="cuda", generator=gen) + 1000
        want = reference(x.double(), groups, torch.ones(c, device="cuda", dtype=torch.float64), torch.zeros(c, device="cuda", dtype=torch.float64), 1e-5, "none",
                         torch.full((n,), s, device="cuda"))["y"][0].reshape(x.shape)
        # x - mean is exact to 1000 half ulps, the mean to a few
        assert (gelib.group_norm_act(x, groups).double() - want).abs().max() < 8 * 1000 * 2.0 ** -24


def test_nothing_and_infinities(gelib):
    for shape in ((0, 3, 8), (3, 0, 8), (0, 8)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        w = torch.ones(8, device="cuda", requires_grad=True)
        y = gelib.group_norm_act(x, 2, w)
        gx, gw = torch.autograd.grad(y.sum(), (x, w))
        assert y.shape == x.shape and gx.shape == x.shape and not gw.any()
    x = torch.randn(3, 50, 16, device="cuda")
    clean = gelib.group_norm_act(x, 4)
    x[1, 7, 5] = float("nan")
    y = gelib.group_norm_act(x, 4)
    assert torch.isnan(y[1, :, 4:8]).all()
    y[1, :, 4:8] = clean[1, :, 4:8]
    assert torch.equal(y, clean)
    # equal values: the difference from the mean is rounding at most, eps holds the rest
    assert gelib.group_norm_act(torch.full((2, 40, 16), 3.0, device="cuda"), 4).abs().max() == 0


def test_differences(gelib):
    """Directional differences of a float32 function: h^2 of the third derivative, and u |y| / h of rounding, both below 2e-3 of the sum."""
    gen = torch.Generator(device="cuda").manual_seed(8)

    def randn(*s):
        return torch.randn(*s, device="cuda", generator=gen)
    for act in ("none", "silu", "gelu"):
        x, w, b, g = randn(3, 21, 24), 1 + 0.1 * randn(24), randn(24), randn(3, 21, 24)
        d = [randn(*t.shape) for t in (x, w, b)]
        ts = [t.clone().requires_grad_() for t in (x, w, b)]
        lengths = torch.tensor([21, 9, 2], device="cuda", dtype=torch.int32)
        f = lambda *t: (gelib.group_norm_act(t[0], 6, t[1], t[2], act=act, lengths=lengths).double() * g).sum()  # noqa: E731
        grads = torch.autograd.grad(f(*ts), ts)
        for k in range(3):
            h = 1e-2
            up, down = ([t + s * h * dk if i == k else t for i, (t, dk) in enumerate(zip((x, w, b), d))] for s in (1, -1))
            slope = (f(*up) - f(*down)) / (2 * h)
            terms = grads[k].double() * d[k]
            assert (slope - terms.sum()).abs() <= 2e-3 * terms.abs().sum(), (act, k)


def test_second_gradients(gelib):
    x = torch.randn(2, 7, 12, device="cuda", requires_grad=True)
    w = torch.randn(12, device="cuda", requires_grad=True)
    lengths = torch.tensor([7, 3], device="cuda", dtype=torch.int32)
    outs = []
    for f in (lambda: gelib.group_norm_act(x, 3, w, act="silu", lengths=lengths),
              lambda: torch.stack([torch.nn.functional.pad(torch.nn.functional.silu(torch.nn.functional.group_norm(
                  x[k:k + 1, :n].transpose(1, 2), 3, w).transpose(1, 2)), (0, 0, 0, 7 - n))[0] for k, n in enumerate((7, 3))])):
        gx, = torch.autograd.grad(f().square().sum(), x, create_graph=True)
        outs.append(torch.autograd.grad(gx.square().sum(), (x, w)))
    for a, b in zip(*outs):
        assert torch.allclose(a, b, rtol=1e-3, atol=1e-3 * float(b.abs().max()))


def test_another_stream_and_graph(gelib):
    x, w = torch.randn(7, 900, 64, device="cuda"), torch.randn(64, device="cuda")
    want = gelib.group_norm_act(x, 8, w, act="gelu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = gelib.group_norm_act(x, 8, w, act="gelu")
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    xs, gs = x.clone(), torch.randn_like(x)
    leaf = xs.requires_grad_()

    def step():
        y = gelib.group_norm_act(leaf, 8, w, act="gelu")
        return (y.detach(), *torch.autograd.grad(y, leaf, gs))   # (no graph outlives a step: its nodes belong to the stream that it was made on)
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        with torch.no_grad():
            leaf.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in out]
        for a, b in zip(kept, step()):
            assert torch.equal(a, b)


def test_refusals(gelib):
    x = torch.randn(2, 5, 12, device="cuda")
    ok = dict(dtype=torch.float32, device="cuda")
    for bad, error in ((lambda: gelib.group_norm_act(x, 5), ValueError), (lambda: gelib.group_norm_act(x, 0), ValueError),
                       (lambda: gelib.group_norm_act(x[0, 0], 1), ValueError), (lambda: gelib.group_norm_act(x.cpu(), 3), ValueError),
                       (lambda: gelib.group_norm_act(x.double(), 3), TypeError), (lambda: gelib.group_norm_act(x, 3, act="tanh"), ValueError),
                       (lambda: gelib.group_norm_act(x, 3, torch.ones(11, **ok)), ValueError), (lambda: gelib.group_norm_act(x, 3, torch.ones(12)), ValueError),
                       (lambda: gelib.group_norm_act(x, 3, torch.ones(12, **ok).half()), TypeError), (lambda: gelib.group_norm_act(x, 3, eps=-1.0), ValueError),
                       (lambda: gelib.group_norm_act(x, 3, lengths=torch.ones(2, device="cuda")), TypeError),
                       (lambda: gelib.group_norm_act(x, 3, lengths=torch.ones(3, device="cuda", dtype=torch.int32)), ValueError),
                       (lambda: gelib.group_norm_act(x, 3, lengths=torch.ones(2, dtype=torch.int32)), ValueError),
                       (lambda: gelib.group_norm_act(x.requires_grad_(), 5), ValueError)):
        with pytest.raises(error):
            bad()
