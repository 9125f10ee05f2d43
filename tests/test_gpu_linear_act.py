"""linear_act and its gradients against the formulas in float64.  Tolerances, u = 2^-24 and h the half ulp of the layer's type: a dot
product of k terms is off by (k + 4) u of the sum of their moduli; act and act' change by 1.2 of a change of z (relu: act' by 1 where z is
within its error of zero); act' is kept to 2^-11 (float16) in 16-bit layers; the gradient that enters the backward products is
rounded to the layer's type (h); results are rounded once."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests.test_gpu_group_norm import HALF_ULP, act64, check, slope64, u  # noqa: E402


@pytest.fixture(scope="module")
def gelib():
    assert torch.cuda.is_available()
    import gelib_amd
    return gelib_amd


def reference(x, w, b, r, act, g, dtype):
    z = x @ w + b
    dz = (x.shape[1] + 4) * u * (x.abs() @ w.abs()) + 4 * u * (z.abs() + b.abs())
    out = {"y": (act64(z, act) + r, 1.2 * dz + 16 * u * z.abs() * (1 + z.abs()) + 2 * u * r.abs())}
    slope = slope64(z, act)
    h = HALF_ULP[dtype]
    rest = 0. if act == "none" else (2.0 ** -11 * slope.abs() + 2.0 ** -25 if dtype != torch.float32 else 0.) + 16 * u * (1 + z.abs())
    dgz = g.abs() * ((torch.where(z.abs() <= dz, 1., 0.) if act == "relu" else (0. if act == "none" else 1.2) * dz) + rest)
    gz = g * slope
    out["gb"] = gz.sum(0), (dgz + (64 + len(g) / 64) * u * gz.abs()).sum(0)
    dgz = dgz + (h * (gz.abs() + dgz) if act != "none" else 0.)
    gx, gw = (dgz @ w.abs().t() + (w.shape[1] + 4) * u * (gz.abs() @ w.abs().t())), x.abs().t() @ dgz + (len(g) + 4) * u * (x.abs().t() @ gz.abs())
    out["gx"], out["gw"] = (gz @ w.t(), gx), (x.t() @ gz, gw)
    return out


# rows, n_in, n_out: one of everything, single rows and columns, sizes around the tiles (16, 64, 128, 256) and their steps, long sums that
# are cut into pieces, odd sizes whose rows are not aligned, an empty sum
SHAPES = [(1, 1, 1), (1, 512, 700), (3, 40, 8), (7, 33, 1), (16, 16, 16), (17, 4099, 65), (64, 64, 64), (65, 63, 129), (128, 256, 128), (129, 72, 257), (300, 1, 5),
          (255, 130, 384), (513, 96, 264), (1000, 8, 40), (5003, 24, 30), (2, 8, 5000), (260, 1024, 520), (5, 0, 6)]
# up to four rows: any columns, k below and above what one batch of loads takes, and the first k that goes to the tiles
SHAPES += [(1, 1024, 256), (1, 2049, 72), (2, 1000, 130), (3, 341, 64), (4, 512, 1040), (4, 100, 3), (1, 7, 4100)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gradients_are_rounded_twice_and_no_more(gelib, act, dtype):
    # Where the layer's type rounds gz and the results and nothing else does, the formulas with these two roundings are as far off; the
    # mean of 10^5 squared errors and more has a spread below 1 %, and the slope adds less than (1/8)^2 to the two squares: 1.03.
    gen = torch.Generator(device="cuda").manual_seed(5)
    x, w, g = (torch.randn(*s, device="cuda", generator=gen).to(dtype) for s in ((900, 320), (320, 410), (900, 410)))
    w = (w / 18).requires_grad_()
    x.requires_grad_()
    got = torch.autograd.grad(gelib.linear_act(x, w, act=act), (x, w), g)
    with torch.no_grad():
        gz = g.double() * slope64(x.double() @ w.double(), act)
        rounded = gz.to(dtype).double()
        for name, v, a, b in (("gx", got[0], (gz @ w.double().t()), rounded @ w.double().t()), ("gw", got[1], x.double().t() @ gz, x.double().t() @ rounded)):
            ours, twice = (v.double() - a).norm(), (b.to(dtype).double() - a).norm()
            assert ours <= 1.03 * twice, (name, float(ours / twice))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("act", ["relu", "silu", "gelu"])
def test_what_is_not_a_number_stays_so_in_gradients(gelib, act, dtype):
    x = torch.ones(40, 24, device="cuda", dtype=dtype)
    x[3, 5] = float("nan")
    x.requires_grad_()
    w = torch.full((24, 16), 0.01, device="cuda", dtype=dtype).requires_grad_()
    gx, gw = torch.autograd.grad(gelib.linear_act(x, w, act=act).float().sum(), (x, w))
    assert torch.isnan(gx[3]).all() and not torch.isnan(gx[[k for k in range(40) if k != 3]]).any() and torch.isnan(gw).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_values_and_gradients(gelib, shape, act, dtype):
    m, k, n = shape
    gen = torch.Generator(device="cuda").manual_seed(m * 7 + k * 3 + n)

    def randn(*size):
        return torch.randn(*size, device="cuda", generator=gen).to(dtype).requires_grad_()
    x, b, r, g = randn(m, k), randn(n), randn(m, n), randn(m, n).detach()
    w = (torch.randn(k, n, device="cuda", generator=gen) / max(k, 1) ** 0.5).to(dtype).requires_grad_()
    y = gelib.linear_act(x, w, b, residual=r, act=act)
    got = dict(zip(("gx", "gw", "gb", "gr"), torch.autograd.grad(y, (x, w, b, r), g)), y=y.detach())
    with torch.no_grad():
        want = reference(x.double(), w.double(), b.double(), r.double(), act, g.double(), dtype)
    for name, (v, tol) in want.items():
        check(got[name], v, tol, "%s of %s" % (name, shape))
    assert torch.equal(got["gr"], g)
    assert torch.equal(y, gelib.linear_act(x.detach(), w.detach(), b.detach(), residual=r.detach(), act=act))
    again = torch.autograd.grad(gelib.linear_act(x, w, b, residual=r, act=act), (x, w, b), g)
    for a, name in zip(again, ("gx", "gw", "gb")):
        assert torch.equal(a, got[name])   # fixed orders of summation
    # each gradient by itself, and without bias and residual
    for some in ((x,), (w,), (b,)):
        a, = torch.autograd.grad(gelib.linear_act(x, w, b, residual=r, act=act), some, g)
        assert torch.equal(a, got[{id(x): "gx", id(w): "gw", id(b): "gb"}[id(some[0])]])
    zero = torch.zeros_like(b), torch.zeros_like(r)
    assert torch.equal(gelib.linear_act(x, w, act=act) + 0, gelib.linear_act(x, w, zero[0], residual=zero[1], act=act) + 0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_layouts(gelib, dtype):
    gen = torch.Generator(device="cuda").manual_seed(5)

    def randn(*s):
        return torch.randn(*s, device="cuda", generator=gen).to(dtype)
    big, W = randn(6, 9, 11, 80), randn(100, 70)
    for x in (big, big[:, :, :, 5:37], big[:, 2:7, :, 8:24], big.transpose(1, 2), big[..., ::2], big[0, 0, 0], big[0, :, 0, 1:33], big[:1, :1, :1, :16].expand(3, 5, 4, 16)):
        for w in (W[:x.shape[-1], :48], W[1:1 + x.shape[-1], 3:36], randn(40, 80)[:, :x.shape[-1]].t()):
            r = randn(*x.shape[:-1], 2 * w.shape[1])[..., ::2]
            outs = []
            for f in (lambda t: t, lambda t: t.contiguous()):
                ts = [f(t).detach().requires_grad_() for t in (x, w, r)]
                y = gelib.linear_act(ts[0], ts[1], residual=ts[2], act="silu")
                outs.append((y, *torch.autograd.grad(y, ts, torch.ones((), device="cuda", dtype=dtype).expand(y.shape))))
            assert y.shape == (*x.shape[:-1], w.shape[1])
            for a, b in zip(*outs):
                assert torch.equal(a, b)


def test_memory_beside_the_operands_is_not_touched_or_read(gelib):
    """Operands between NaNs, and results between sentinels, through the C ABI: the tiles' ragged ends stay inside."""
    from gelib_amd import cabi
    import ctypes
    L = cabi.lib()
    vp = ctypes.c_void_p
    for dtype, code in ((torch.float32, 0), (torch.bfloat16, 1)):
        for m, k, n in ((1, 40, 72), (17, 33, 65), (130, 100, 257), (300, 520, 40), (4, 2000, 24)):
            def framed(rows, cols, fill=None):
                t = torch.full((rows * cols + 1024,), float("nan"), device="cuda", dtype=dtype)
                inner = t[512:512 + rows * cols].view(rows, cols)
                if fill is None:
                    inner.normal_()
                return t, inner
            (X, x), (W, w), (G, g) = framed(m, k), framed(k, n), framed(m, n)
            (Y, y), (GX, gx), (GW, gw) = framed(m, n, 0), framed(m, k, 0), framed(k, n, 0)
            stream = vp(torch.cuda.current_stream().cuda_stream)
            need = int(L.gelib_hip_linear_act_workspace_bytes(0, code, m, k, n))
            ws = torch.full((max(need, 16),), 255, device="cuda", dtype=torch.uint8)
            cabi.check(L.gelib_hip_linear_act_fwd(vp(y.data_ptr()), None, vp(x.data_ptr()), vp(w.data_ptr()), None, None, code, ctypes.c_int64(m), k, n,
                                                  ctypes.c_int64(k), 0, vp(ws.data_ptr()), ctypes.c_uint64(need), stream))
            need = int(L.gelib_hip_linear_act_workspace_bytes(3, code, m, k, n))
            ws = torch.full((max(need, 16),), 255, device="cuda", dtype=torch.uint8)
            cabi.check(L.gelib_hip_linear_act_bwd(vp(gx.data_ptr()), vp(gw.data_ptr()), None, vp(g.data_ptr()), None, vp(x.data_ptr()), vp(w.data_ptr()), code,
                                                  ctypes.c_int64(m), k, n, ctypes.c_int64(k), vp(ws.data_ptr()), ctypes.c_uint64(need), stream))
            want = reference(x.double(), w.double(), torch.zeros(n, device="cuda", dtype=torch.float64), torch.zeros(m, n, device="cuda", dtype=torch.float64),
                             "none", g.double(), dtype)
            for got, name in ((y, "y"), (gx, "gx"), (gw, "gw")):
                check(got, *want[name], "%s of %s" % (name, (m, k, n)))
            for t in (Y, GX, GW):
                assert torch.isnan(t[:512]).all() and torch.isnan(t[-512:]).all()


def test_offsets_beyond_32_bits(gelib):
    """4.4 GB of x and 4.6 of the result: the last rows are what they are by themselves."""
    m, k, n = 1050000, 2056, 2100
    x = torch.zeros(m, k, device="cuda", dtype=torch.bfloat16)
    x[-70:] = torch.randn(70, k, device="cuda")
    w, b = (torch.randn(k, n, device="cuda") / 50).bfloat16(), torch.randn(n, device="cuda").bfloat16()
    y = gelib.linear_act(x, w, b, residual=torch.zeros(1, 1, device="cuda", dtype=torch.bfloat16).expand(m, n), act="relu")
    want = reference(x[-70:].double(), w.double(), b.double(), torch.zeros(70, n, device="cuda", dtype=torch.float64), "relu",
                     torch.zeros(70, n, device="cuda", dtype=torch.float64), torch.bfloat16)["y"]
    check(y[-70:], *want, "the last rows")
    assert torch.equal(y[:5], b.clamp(min=0).expand(5, n)) and torch.equal(y[m // 2], b.clamp(min=0))
    del y
    x.requires_grad_()
    w.requires_grad_()
    g = torch.zeros(m, n, device="cuda", dtype=torch.bfloat16)
    g[-70:] = torch.randn(70, n, device="cuda")
    gx, gw = torch.autograd.grad(gelib.linear_act(x, w, b, act="none"), (x, w), g)
    zero = torch.zeros(70, n, device="cuda", dtype=torch.float64)
    want = reference(x[-70:].detach().double(), w.detach().double(), b.double(), zero, "none", g[-70:].double(), torch.bfloat16)
    check(gx[-70:], *want["gx"], "gx")
    check(gw, want["gw"][0], want["gw"][1] + 64 * u * want["gw"][0].abs(), "gw")   # (the other rows add zeros)
    assert not gx[:-70].any()


def test_infinities_stay_in_their_rows_and_columns(gelib):
    for dtype in (torch.float32, torch.bfloat16):
        for m, k, n in ((40, 96, 130), (300, 260, 200), (2, 520, 136)):
            x, w = torch.randn(m, k, device="cuda").to(dtype), torch.randn(k, n, device="cuda").to(dtype)
            clean = gelib.linear_act(x, w, act="silu")
            x[1, 3] = float("nan")
            y = gelib.linear_act(x, w, act="silu")
            assert torch.isnan(y[1]).all()
            y[1] = clean[1]
            assert torch.equal(y, clean)


def test_nothing(gelib):
    w = torch.randn(8, 6, device="cuda", requires_grad=True)
    b = torch.randn(6, device="cuda", requires_grad=True)
    x = torch.zeros(0, 8, device="cuda", requires_grad=True)
    y = gelib.linear_act(x, w, b, act="silu")
    gx, gw, gb = torch.autograd.grad(y.sum(), (x, w, b))
    assert y.shape == (0, 6) and gx.shape == (0, 8) and not gw.any() and not gb.any()
    assert gelib.linear_act(torch.zeros(4, 8, device="cuda"), torch.zeros(8, 0, device="cuda")).shape == (4, 0)


def test_differences(gelib):
    """Directional differences of a float32 function: h^2 of the third derivative, and u |y| / h of rounding, both below 2e-3 of the sum."""
    gen = torch.Generator(device="cuda").manual_seed(8)

    def randn(*s):
        return torch.randn(*s, device="cuda", generator=gen)
    for act in ("none", "silu", "gelu"):
        ts, g = (randn(33, 20), randn(20, 18) / 4, randn(18), randn(33, 18)), randn(33, 18)
        d = [randn(*t.shape) for t in ts]
        leaves = [t.clone().requires_grad_() for t in ts]
        f = lambda x, w, b, r: (gelib.linear_act(x, w, b, residual=r, act=act).double() * g).sum()  # noqa: E731
        grads = torch.autograd.grad(f(*leaves), leaves)
        for k in range(4):
            h = 1e-2
            up, down = ([t + s * h * dk if i == k else t for i, (t, dk) in enumerate(zip(ts, d))] for s in (1, -1))
            terms = grads[k].double() * d[k]
            assert ((f(*up) - f(*down)) / (2 * h) - terms.sum()).abs() <= 2e-3 * terms.abs().sum(), (act, k)


def test_second_gradients(gelib):
    x, w, b, r = (torch.randn(*s, device="cuda", requires_grad=True) for s in ((9, 12), (12, 5), (5,), (9, 5)))
    outs = []
    for f in (lambda: gelib.linear_act(x, w, b, residual=r, act="silu"), lambda: torch.nn.functional.silu(x @ w + b) + r):
        gx, gw = torch.autograd.grad(f().square().sum(), (x, w), create_graph=True)
        outs.append(torch.autograd.grad(gx.square().sum() + gw.sum(), (x, w, b, r)))
    for p, q in zip(*outs):
        assert torch.allclose(p, q, rtol=1e-3, atol=1e-3 * float(q.abs().max()))


def test_another_stream_and_graph(gelib):
    ts = [torch.randn(300, 200, device="cuda").bfloat16().requires_grad_(), torch.randn(200, 90, device="cuda").bfloat16().requires_grad_(),
          torch.randn(90, device="cuda").bfloat16().requires_grad_()]
    g = torch.randn(300, 90, device="cuda").bfloat16()

    def step():
        y = gelib.linear_act(*ts, act="gelu")
        return (y.detach(), *torch.autograd.grad(y, ts, g))   # (no graph outlives a step: its nodes belong to the stream that it was made on)
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        with torch.no_grad():
            ts[0].copy_(torch.randn(300, 200, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in out]
        for a, b in zip(kept, step()):
            assert torch.equal(a, b)


def test_refusals(gelib):
    x, w = torch.randn(4, 8, device="cuda"), torch.randn(8, 6, device="cuda")
    b, r = torch.randn(6, device="cuda"), torch.randn(4, 6, device="cuda")
    for bad, error in ((lambda: gelib.linear_act(x, w[:7]), ValueError), (lambda: gelib.linear_act(x, w[0]), ValueError), (lambda: gelib.linear_act(x.cpu(), w), ValueError),
                       (lambda: gelib.linear_act(x, w.cpu()), ValueError), (lambda: gelib.linear_act(x.half(), w), TypeError),
                       (lambda: gelib.linear_act(x.double(), w.double()), TypeError), (lambda: gelib.linear_act(x, w, b[:5]), ValueError),
                       (lambda: gelib.linear_act(x, w, b.half()), TypeError), (lambda: gelib.linear_act(x, w, b, residual=r[:3]), ValueError),
                       (lambda: gelib.linear_act(x, w, b, residual=b), ValueError), (lambda: gelib.linear_act(x, w, b, act="tanh"), ValueError),
                       (lambda: gelib.linear_act(x, w.clone().requires_grad_(), b.cpu()), ValueError)):
        with pytest.raises(error):
            bad()
