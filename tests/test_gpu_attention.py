"""attention and its gradients against the formulas in float64, document by document.  Tolerances, u = 2^-24 and h the half ulp of the
type: a score is off by (dim + 4) u of the sum of the moduli of its products, and its distance's term by 8 u (differences, squares, root,
slope, product); the hardware's exponential and logarithm by 2 u; so a weight p is relatively off by twice the largest of its row's scores'
errors plus (keys + 16) u, and by h where it is rounded for the product with v.  gy . v is off by (dim + 4) u of its moduli, D by what y is off,
rounded to its type, times |gy|; ds = p (gy . v - D) by the two together, and by h in 16 bits; the gradients are sums of these
products, off by (terms + 8) u of their moduli besides.  Results are rounded once (in check).  Errors of sums of scaled values down to the
smallest: LEAST of the type, for every term of a sum that float16 rounds."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests.test_gpu_group_norm import HALF_ULP, LEAST, check, u  # noqa: E402


@pytest.fixture(scope="module")
def gelib():
    assert torch.cuda.is_available()
    import gelib_amd
    return gelib_amd


def document(q, k, v, x, xk, slopes, g, scale, dtype):
    """One document: {name: (value, tolerance)}.  q, g (nq, heads, dim), k, v (nk, kv heads, dim), all float64."""
    nq, H, dim = q.shape
    nk, KV = k.shape[:2]
    h = 0. if dtype == torch.float32 else HALF_ULP[dtype]
    least = 0. if dtype == torch.float32 else LEAST[dtype]
    kk, vv = (t.repeat_interleave(H // KV, 1).transpose(0, 1) for t in (k, v))     # (heads, nk, dim)
    qq, gg = q.transpose(0, 1), g.transpose(0, 1)
    s = scale * qq @ kk.transpose(1, 2)
    es = abs(scale) * (dim + 4) * u * (qq.abs() @ kk.abs().transpose(1, 2))
    if slopes is not None:
        apart = x[:, None] - xk[None]
        far = apart.square().sum(2).sqrt()
        s = s - slopes[:, None, None] * far
        es = es + 8 * u * slopes.abs()[:, None, None] * far
    es = es + 4 * u * s.abs()
    if nk:
        p = torch.softmax(s, 2)
        rel = 2 * es.amax(2, keepdim=True) + (nk + 16) * u
        few = 2.0 ** -140
    else:
        p, rel, few = s, s.sum(2, keepdim=True), 0.
    out = {}
    y = p @ vv
    ey = (p * (rel + h) + few + least) @ vv.abs() + (nk + 8) * u * (p @ vv.abs())
    out["y"] = y.transpose(0, 1), ey.transpose(0, 1)
    eround = ey + (HALF_ULP[dtype] * y.abs() + LEAST[dtype])
    dp = gg @ vv.transpose(1, 2)
    edp = (dim + 4) * u * (gg.abs() @ vv.abs().transpose(1, 2))
    D = (gg * y).sum(2, keepdim=True)
    eD = (gg.abs() * eround).sum(2, keepdim=True) + (dim + 4) * u * (gg * y).abs().sum(2, keepdim=True)
    ds = p * (dp - D)
    eds = p * rel * (dp - D).abs() + p * (edp + eD) + 4 * u * ds.abs() + few
    e16 = eds + h * (ds.abs() + eds) + least
    out["gq"] = (scale * ds @ kk).transpose(0, 1), (abs(scale) * (e16 + (nk + 8) * u * ds.abs()) @ kk.abs()).transpose(0, 1)

    def group(t):
        return t.unflatten(0, (KV, H // KV)).sum(1).transpose(0, 1)
    terms = nq * H // KV + 8
    out["gk"] = group(scale * ds.transpose(1, 2) @ qq), group(abs(scale) * (e16 + terms * u * ds.abs()).transpose(1, 2) @ qq.abs())
    out["gv"] = group(p.transpose(1, 2) @ gg), group((p * (rel + h + terms * u) + few + least).transpose(1, 2) @ gg.abs())
    if slopes is not None:
        out["gslopes"] = -(ds * far).sum((1, 2)), ((eds + (nk + nq + 32) * u * ds.abs()) * far).sum((1, 2))
        w = slopes[:, None, None]
        each = ((ds * w)[..., None] * apart / far.masked_fill(far == 0, 1)[..., None]).sum(0)          # (nq, nk, 3)
        unit = (apart / far.masked_fill(far == 0, 1)[..., None]).abs()
        tol = (((eds + (nk + nq + 32) * u * ds.abs()) * w.abs()).sum(0)[..., None] * (unit + 8 * u)) + 8 * u * (ds * w).abs().sum(0)[..., None]
        out["gx"] = -each.sum(1), tol.sum(1)
        out["gxk"] = each.sum(0), tol.sum(0)
    return out


def compare(gelib, dtype, docs, heads, kv, dim, packed, geometry=True, same=True, seed=0, scale=None, spoil=False, every=True):
    """docs: [(queries, keys)], as packed documents (with rows in none around them) or padded to the largest (and one more)."""
    gen = torch.Generator(device="cuda").manual_seed(seed + dim * 7 + heads)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)
    n = len(docs)
    if packed:
        qs, ks = [2], [2 if same else 1]
        for a, b in docs:
            qs.append(qs[-1] + a)
            ks.append(ks[-1] + b)
        nq, nk = qs[-1] + 3, ks[-1] + (3 if same else 5)
        shape_q, shape_k = (nq,), (nk,)
        where = [((slice(a, b),), (slice(c, d),)) for a, b, c, d in zip(qs, qs[1:], ks, ks[1:])]
        masks = dict(starts=torch.tensor(ks, device="cuda", dtype=torch.int32))
        if not same:
            masks["query_starts"] = torch.tensor(qs, device="cuda", dtype=torch.int32)
    else:
        nq, nk = max(a for a, _ in docs) + 1, max(b for _, b in docs) + 1
        shape_q, shape_k = (n, nq), (n, nk)
        where = [((d, slice(0, a)), (d, slice(0, b))) for d, (a, b) in enumerate(docs)]
        masks = dict(lengths=torch.tensor([b for _, b in docs], device="cuda", dtype=torch.int32),
                     query_lengths=torch.tensor([a for a, _ in docs], device="cuda", dtype=torch.int32))
    q, k, v, g = randn(*shape_q, heads, dim).to(dtype), randn(*shape_k, kv, dim).to(dtype), randn(*shape_k, kv, dim).to(dtype), randn(*shape_q, heads, dim).to(dtype)
    x = xk = slopes = None
    if geometry:
        x = randn(*shape_q, 3) * 2 + 5
        xk = x if same else randn(*shape_k, 3) * 2 + 5
        slopes = torch.rand(heads, device="cuda", generator=gen) + 0.05
    if spoil:   # what does not exist may be anything
        gone_q, gone_k = torch.ones(shape_q, dtype=torch.bool, device="cuda"), torch.ones(shape_k, dtype=torch.bool, device="cuda")
        for a, b in where:
            gone_q[a], gone_k[b] = False, False
        q[gone_q], k[gone_k], v[gone_k], g[gone_q] = float("nan"), float("inf"), float("nan"), float("-inf")
        if geometry:
            x[gone_q & gone_k if same else gone_q] = float("nan")
            xk[gone_q & gone_k if same else gone_k] = float("nan")
    leaves = {"gq": q, "gk": k, "gv": v}
    if geometry:
        leaves.update({"gx": x, "gslopes": slopes}, **({} if same else {"gxk": xk}))
    for t in leaves.values():
        t.requires_grad_()
    y = gelib.attention(q, k, v, x, slopes, key_points=None if same else xk, scale=scale, **masks)
    got = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), g)), y=y.detach())
    c = dim ** -0.5 if scale is None else scale
    zero = {name: torch.zeros(t.shape, device="cuda", dtype=torch.float64) for name, t in dict(leaves, y=q).items()}
    want, tol = zero, {name: t.clone() for name, t in zero.items()}
    with torch.no_grad():
        for a, b in where:
            one = document(q[a].double(), k[b].double(), v[b].double(), *((x[a].double(), xk[b].double(), slopes.double()) if geometry else (None, None, None)),
                           g[a].double(), c, dtype)
            if same and geometry:
                one["gx"] = one["gx"][0] + one["gxk"][0], one["gx"][1] + one["gxk"][1]
            for name in want:
                at = b if name in ("gk", "gv", "gxk") else (slice(None),) if name == "gslopes" else a
                want[name][at] += one[name][0]
                tol[name][at] += one[name][1]
    for name in want:
        check(got[name], want[name], tol[name], "%s of %s, %s heads of %s" % (name, docs, heads, dim))
    assert torch.equal(y, gelib.attention(*(t.detach() if t is not None else None for t in (q, k, v, x, slopes)), key_points=None if same else xk.detach() if geometry else None,
                                          scale=scale, **masks))
    if every:   # the same bits again, and each gradient by itself
        again = torch.autograd.grad(gelib.attention(q, k, v, x, slopes, key_points=None if same else xk, scale=scale, **masks), list(leaves.values()), g)
        for name, t in zip(leaves, again):
            assert torch.equal(t, got[name]), name
        for name, leaf in leaves.items():
            one, = torch.autograd.grad(gelib.attention(q, k, v, x, slopes, key_points=None if same else xk, scale=scale, **masks), leaf, g)
            assert torch.allclose(one.float(), got[name].float(), rtol=0.02, atol=1e-3 * float(got[name].float().abs().max())), name


TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("packed", [False, True], ids=["padded", "packed"])
@pytest.mark.parametrize("dim", [1, 8, 17, 32, 40, 64, 72, 100, 128])
def test_sizes_of_heads(gelib, dim, packed, dtype):
    compare(gelib, dtype, [(19, 19), (1, 1), (0, 0), (33, 33)], 4, 2, dim, packed)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("packed", [False, True], ids=["padded", "packed"])
@pytest.mark.parametrize("heads,kv", [(1, 1), (8, 8), (7, 1), (6, 2), (16, 4)])
def test_heads(gelib, heads, kv, packed, dtype):
    compare(gelib, dtype, [(5, 5), (16, 16), (40, 40), (0, 0), (1, 1)], heads, kv, 24, packed)


# around the tiles: 16 rows, 32 and 128 of a block, 64 (or 32) of the other side; documents that fill a block and ones that do not
LENGTHS = [[(1, 1)], [(2, 2), (15, 15), (16, 16), (17, 17)], [(31, 31), (32, 32), (33, 33)], [(63, 63), (64, 64), (65, 65), (0, 0), (0, 0)], [(127, 127), (128, 128), (129, 129)],
           [(300, 300), (5, 5)], [(0, 0)], [(1000, 1000)]]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("packed", [False, True], ids=["padded", "packed"])
@pytest.mark.parametrize("docs", LENGTHS, ids=lambda d: "-".join(str(a) for a, _ in d))
def test_lengths(gelib, docs, packed, dtype):
    compare(gelib, dtype, docs, 3, 3, 32, packed, spoil=True)


# queries and keys that are not the same rows; a query without keys, keys without a query, single queries over many keys (which are cut
# into pieces), many queries of a few keys
CROSS = [[(1, 40), (3, 0), (0, 7), (20, 65)], [(1, 2000)], [(1, 700), (1, 3), (1, 0), (1, 1500)], [(600, 3)], [(700, 1), (2, 300)], [(70, 200), (200, 70)]]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("packed", [False, True], ids=["padded", "packed"])
@pytest.mark.parametrize("docs", CROSS, ids=lambda d: "-".join("%dx%d" % p for p in d))
@pytest.mark.parametrize("geometry", [False, True], ids=["plain", "points"])
def test_queries_of_other_keys(gelib, geometry, docs, packed, dtype):
    compare(gelib, dtype, docs, 4, 2, 64, packed, geometry=geometry, same=False, spoil=True)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim", [16, 32, 64, 128])
@pytest.mark.parametrize("heads,kv", [(4, 2), (3, 3), (4, 1), (8, 1), (3, 1)])
def test_long(gelib, heads, kv, dim, dtype):
    """Groups of two, four and eight heads, whose tiles share distances, and others."""
    compare(gelib, dtype, [(1100, 1100), (300, 300)], heads, kv, dim, True, every=False)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("heads,kv", [(3, 3), (4, 2)])
@pytest.mark.parametrize("dim", [16, 32, 64, 128])
def test_long_without_points(gelib, dim, heads, kv, dtype):
    compare(gelib, dtype, [(600, 600), (300, 300)], heads, kv, dim, False, geometry=False, every=False)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim", [16, 32, 64, 128])
def test_many_short_documents(gelib, dim, dtype):
    """So many that a wave takes several heads, one after the other."""
    gen = torch.Generator().manual_seed(3)
    docs = [(k, k) for k in torch.randint(0, 40, (700,), generator=gen).tolist()]
    for packed in (True, False):
        compare(gelib, dtype, docs, 14, 7, dim, packed, every=False)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_far_apart_scores(gelib, dtype):
    """Rows whose maximum grows through many tiles, and scores that leave one key with everything."""
    compare(gelib, dtype, [(200, 900)], 2, 1, 32, False, same=False, scale=-3.0, every=False)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_no_masks(gelib, dtype):
    """No lengths at all, and lengths beyond the rows there are, are all rows."""
    q, k, v = (torch.randn(3, n, 4, 32, device="cuda").to(dtype) for n in (20, 50, 50))
    many = torch.full((3,), 1 << 30, device="cuda", dtype=torch.int32)
    y = gelib.attention(q, k, v)
    assert torch.equal(y, gelib.attention(q, k, v, lengths=many, query_lengths=many))
    none = torch.full((3,), -5, device="cuda", dtype=torch.int32)
    assert (gelib.attention(q, k, v, lengths=none) == 0).all() and (gelib.attention(q, k, v, query_lengths=none) == 0).all()
    one = gelib.attention(q.view(60, 4, 32), k.reshape(150, 4, 32), v.reshape(150, 4, 32), starts=torch.tensor([0, 50, 100, 150], device="cuda", dtype=torch.int32),
                          query_starts=torch.tensor([0, 20, 40, 60], device="cuda", dtype=torch.int32))
    assert torch.equal(one.view(3, 20, 4, 32), y)


def test_starts_outside_of_the_rows(gelib):
    """Starts are held to the rows there are; whatever they say, nothing outside is read, and documents in order are right."""
    q = torch.randn(40, 2, 32, device="cuda")

    def call(starts):
        return gelib.attention(q, q, q, starts=torch.tensor(starts, device="cuda", dtype=torch.int32))
    assert torch.equal(call([-7, 20, 1 << 30]), call([0, 20, 40]))
    assert (call([0]) == 0).all() and (call([5, 5, 5]) == 0).all()
    for bad in ([40, 0], [30, 10, 20, 5], [1 << 30, -1 << 30, 12]):
        call(bad)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_layouts(gelib, dtype):
    """Columns of one layer's result, heads before positions, one head for all, offsets that no wide load takes."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    qkv = torch.randn(3, 30, 8, 41, device="cuda", generator=gen).to(dtype)
    # (float32 strides of 41 values are no multiple of 16 bytes either)
    for q, k, v in ((qkv[:, :, :4, :32], qkv[:, :, 4:6, :32], qkv[:, :, 6:, :32]), (qkv[..., 1:33], qkv[..., 3:35], qkv[..., 5:37]),
                    (qkv[:, :, :4, :16].transpose(0, 1), qkv[:, :, 4:, :16].transpose(0, 1), qkv[:, :, :4, 20:36].transpose(0, 1)),
                    (qkv[:, :, :2, ::2], qkv[:, :, 2:4, ::2], qkv[:, :, 4:6, ::2]), (qkv[:, :, :6], qkv[:, :, :1].expand(3, 30, 6, 41), qkv[:1, :, 2:8].expand(3, 30, 6, 41)),
                    (qkv[..., :32].permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3), qkv[..., :32], qkv[..., :32])):
        x = torch.randn(*q.shape[:2], 3, device="cuda", generator=gen)
        slopes = torch.rand(q.shape[2], device="cuda", generator=gen)
        g = torch.randn(q.shape, device="cuda", generator=gen).to(dtype)
        outs = []
        for f in (lambda t: t, lambda t: t.contiguous()):
            ts = [f(t).detach().requires_grad_() for t in (q, k, v, x, slopes)]
            y = gelib.attention(*ts)
            outs.append((y, *torch.autograd.grad(y, ts, f(g.transpose(0, 1).contiguous().transpose(0, 1)))))
        assert outs[0][0].is_contiguous()
        for a, b in zip(*outs):
            assert torch.equal(a, b)


def test_offsets_beyond_32_bits(gelib):
    """Rows further than 2^31 and 2^32 bytes and elements from the first one (strides), only few of which exist."""
    base = torch.empty((1 << 32) + (1 << 20), device="cuda", dtype=torch.bfloat16)
    far = base.as_strided((5, 2, 32), ((1 << 30), 64, 1))
    gen = torch.Generator(device="cuda").manual_seed(5)
    near = torch.randn(5, 2, 32, device="cuda", generator=gen).bfloat16()
    far.copy_(near)
    starts = torch.tensor([0, 3, 5], device="cuda", dtype=torch.int32)
    ts, us = [far.detach().requires_grad_() for _ in range(3)], [near.detach().clone().requires_grad_() for _ in range(3)]
    a, b = gelib.attention(*ts, starts=starts), gelib.attention(*us, starts=starts)
    assert torch.equal(a, b)
    for s, t in zip(torch.autograd.grad(a, ts, near), torch.autograd.grad(b, us, near)):
        assert torch.equal(s, t)


def test_what_is_not_finite(gelib):
    """NaN in a query stays in its row, NaN in a key in its document; a score of -infinity is a key that has no share."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    q, k, v = (torch.randn(60, 2, 32, device="cuda", generator=gen) for _ in range(3))
    starts = torch.tensor([0, 20, 60], device="cuda", dtype=torch.int32)
    q[5, 1, 3] = float("nan")
    y = gelib.attention(q, k, v, starts=starts)
    bad = torch.zeros(60, 2, dtype=torch.bool, device="cuda")
    bad[5, 1] = True
    assert torch.isnan(y[bad]).all() and torch.isfinite(y[~bad]).all()
    q[5, 1, 3] = 0
    v[30, 0, 7] = float("inf")
    y = gelib.attention(q, k, v, starts=starts)
    assert torch.isfinite(y[:20]).all() and torch.isfinite(y[:, 1]).all() and not torch.isfinite(y[20:, 0, 7]).any()
    v[30, 0, 7] = 0
    q[:], k[:, :, 0] = 0, 0
    q[:, :, 0] = 1
    k[10, :, 0] = float("-inf")
    y = gelib.attention(q, k, v, starts=starts)
    rest = [j for j in range(20) if j != 10]
    assert torch.allclose(y[:20], v[rest].mean(0).expand(20, 2, 32), atol=1e-5)


def test_points_in_one_place(gelib):
    """A distance of zero has no direction: gradients of points are finite, and those of a document of one place zero."""
    q, k, v = (torch.randn(1, 10, 2, 8, device="cuda", requires_grad=True) for _ in range(3))
    x = torch.full((1, 10, 3), 7.25, device="cuda", requires_grad=True)
    slopes = torch.ones(2, device="cuda", requires_grad=True)
    gx, gs = torch.autograd.grad(gelib.attention(q, k, v, x, slopes).square().sum(), (x, slopes))
    assert (gx == 0).all() and (gs == 0).all()


def test_against_differences(gelib):
    """Along a direction, the gradient times it is the slope of the sum: central differences over 2^-7 in float32, 1 % of the sum of moduli
    (third derivatives over 2^-14 / 6, rounding 2^-24 n / 2^-6)."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    q, k, v = (torch.randn(2, 12, 4, 16, device="cuda", generator=gen) for _ in range(3))
    x, slopes = torch.randn(2, 12, 3, device="cuda", generator=gen) * 2, torch.rand(4, device="cuda", generator=gen)
    lengths = torch.tensor([12, 7], device="cuda", dtype=torch.int32)
    ts = [t.requires_grad_() for t in (q, k, v, x, slopes)]
    g = torch.randn(2, 12, 4, 16, device="cuda", generator=gen)

    def f(*args):
        return (gelib.attention(*args, lengths=lengths, query_lengths=lengths).double() * g.double()).sum()
    grads = torch.autograd.grad(f(*ts), ts)
    for i, t in enumerate(ts):
        d = torch.randn(t.shape, device="cuda", generator=gen)
        d /= d.norm()
        with torch.no_grad():
            plus, minus = ([s + e * d if j == i else s for j, s in enumerate(ts)] for e in (2.0 ** -7, -2.0 ** -7))
            slope = (f(*plus) - f(*minus)) / 2.0 ** -6
        assert abs(float(slope - (grads[i].double() * d).sum())) <= 1e-2 * float(grads[i].norm()) + 1e-3, i


@pytest.mark.parametrize("packed", [False, True], ids=["padded", "packed"])
def test_twice(gelib, packed):
    """Gradients of gradients against differences of gradients."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    shape = (11,) if packed else (2, 6)
    q, k, v = (torch.randn(*shape, 2, 8, device="cuda", generator=gen) for _ in range(3))
    x, slopes = torch.randn(*shape, 3, device="cuda", generator=gen) * 2, torch.rand(2, device="cuda", generator=gen)
    mark = torch.tensor([0, 6, 10] if packed else [6, 4], device="cuda", dtype=torch.int32)
    masks = dict(starts=mark) if packed else dict(lengths=mark, query_lengths=mark)
    ts = [t.requires_grad_() for t in (q, k, v, x, slopes)]

    def grads(args, **kw):
        return torch.autograd.grad(gelib.attention(*args, **masks).square().sum(), args, **kw)
    first, graph = grads(ts), grads(ts, create_graph=True)
    for a, b in zip(first, graph):
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-5)
    ds = [torch.randn(t.shape, device="cuda", generator=gen) for t in ts]
    second = torch.autograd.grad(sum((a * d).sum() for a, d in zip(graph, ds)), ts)
    for i, t in enumerate(ts):
        d = torch.randn(t.shape, device="cuda", generator=gen)
        d /= d.norm()
        near = [[(s + e * d).detach().requires_grad_() if j == i else s for j, s in enumerate(ts)] for e in (2.0 ** -7, -2.0 ** -7)]
        plus, minus = (sum((a.double() * c.double()).sum() for a, c in zip(grads(n), ds)) for n in near)
        assert abs(float((plus - minus) / 2.0 ** -6 - (second[i].double() * d).sum())) <= 2e-2 * float(second[i].norm()) + 5e-3, i


def test_another_stream_and_graph(gelib):
    ts = [torch.randn(2, 300, h, 32, device="cuda").bfloat16().requires_grad_() for h in (4, 2, 2)]
    ts += [(torch.randn(2, 300, 3, device="cuda") * 3).requires_grad_(), torch.rand(4, device="cuda").requires_grad_()]
    g = torch.randn(2, 300, 4, 32, device="cuda").bfloat16()
    lengths = torch.tensor([300, 170], device="cuda", dtype=torch.int32)

    def step():
        y = gelib.attention(*ts, lengths=lengths)
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
            ts[0].copy_(torch.randn(2, 300, 4, 32, device="cuda"))
            lengths.copy_(torch.tensor([300 - 50 * k, 20 * k], device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in out]
        for a, b in zip(kept, step()):
            assert torch.equal(a, b)


def test_refusals(gelib):
    q, k = torch.randn(2, 5, 4, 8, device="cuda"), torch.randn(2, 7, 2, 8, device="cuda")
    x, xk, s = torch.randn(2, 5, 3, device="cuda"), torch.randn(2, 7, 3, device="cuda"), torch.rand(4, device="cuda")
    n = torch.tensor([1, 2], device="cuda", dtype=torch.int32)
    p, st = torch.randn(10, 4, 8, device="cuda"), torch.tensor([0, 4, 10], device="cuda", dtype=torch.int32)
    f = gelib.attention
    for bad, error in ((lambda: f(q, k, k[:, :6]), ValueError), (lambda: f(q, k[:1], k[:1]), ValueError), (lambda: f(q, k[..., :7], k[..., :7]), ValueError),
                       (lambda: f(q[:, :, :3], k, k), ValueError), (lambda: f(q, k.half(), k), TypeError), (lambda: f(q, k, k.half()), TypeError), (lambda: f(q, k.cpu(), k), ValueError),
                       (lambda: f(q.double(), k.double(), k.double()), TypeError), (lambda: f(q[0, 0], k[0, 0], k[0, 0]), ValueError), (lambda: f(q, k, k, x), ValueError),
                       (lambda: f(q, k, k, None, s), ValueError), (lambda: f(q, k, k, x, s), ValueError), (lambda: f(q, k, k, x, s[:3], xk), ValueError),
                       (lambda: f(q, k, k, x.double(), s, xk), TypeError), (lambda: f(q, k, k, x, s.half(), xk), TypeError), (lambda: f(q, k, k, x[..., :2], s, xk), ValueError),
                       (lambda: f(q, k, k, x, s, xk[:, :6]), ValueError), (lambda: f(q, k, k, lengths=n.long()), TypeError), (lambda: f(q, k, k, lengths=n[:1]), ValueError),
                       (lambda: f(q, k, k, query_lengths=n.cpu()), ValueError), (lambda: f(q, k, k, starts=st), ValueError), (lambda: f(p, p, p), ValueError),
                       (lambda: f(p, p, p, lengths=n, starts=st), ValueError), (lambda: f(p, p[:9], p[:9], starts=st), ValueError), (lambda: f(p, p, p, starts=st, query_starts=st[:2]), ValueError),
                       (lambda: f(p, p, p, starts=st[:0]), ValueError), (lambda: f(q, k, k, scale=float("inf")), ValueError), (lambda: f(q, k, k, key_points=xk), ValueError),
                       (lambda: f(*(torch.randn(1, 2, 1, 129, device="cuda") for _ in range(3))), ValueError), (lambda: f(*(torch.randn(1, 2, 1, 0, device="cuda") for _ in range(3))), ValueError)):
        with pytest.raises(error):
            bad()


def test_nothing(gelib):
    for nq, nk in ((0, 5), (5, 0), (0, 0)):
        q, k, v = (torch.randn(2, n, 2, 8, device="cuda", requires_grad=True) for n in (nq, nk, nk))
        y = gelib.attention(q, k, v)
        assert y.shape == q.shape and (y == 0).all()
        for t, leaf in zip(torch.autograd.grad(y, (q, k, v), torch.ones_like(y)), (q, k, v)):
            assert t.shape == leaf.shape and (t == 0).all()
    q = torch.randn(0, 4, 2, 8, device="cuda")
    assert gelib.attention(q, q, q).shape == q.shape
