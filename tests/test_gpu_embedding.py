"""embedding and the gradient of its table against the definition in float64.  Tolerances, u = 2^-24: a value is one product in float32,
a gradient a float32 sum, in pieces, of the gradients of one token (at most tokens additions one after the other) and one product: off by
(n + 2) u of the sum of their moduli, n the tokens of that row; results are rounded once (in check)."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests.test_gpu_group_norm import check, u  # noqa: E402


@pytest.fixture(scope="module")
def gelib():
    assert torch.cuda.is_available()
    import gelib_amd
    return gelib_amd


def reference(tokens, table, g, scale):
    rows = len(table)
    t = tokens.reshape(-1).long()
    ok = (t >= 0) & (t < rows)
    at = t.clamp(0, max(rows - 1, 0))
    y = torch.where(ok[:, None], table[at] * scale, 0.)
    zero = torch.zeros_like(table)
    moduli = zero.index_add(0, at[ok], g[ok].abs())
    return y, zero.index_add(0, at[ok], g[ok]) * scale, (torch.bincount(at[ok], minlength=rows)[:, None] + 2) * u * moduli * abs(scale)


# tokens, rows, channels: one of everything, sizes around pieces (32, 64, 128 tokens), a block's 2048, and a digit's 256 rows; widths of one to
# many loads, aligned or not; one row for all tokens, mostly rows without one
SIZES = [(1, 1, 1), (1, 5, 8), (3, 2, 7), (31, 4, 16), (32, 1, 64), (33, 1, 65), (64, 256, 24), (65, 257, 130), (2047, 300, 33), (2048, 118, 64), (2049, 1, 128), (5000, 70000, 40),
         (16384, 3, 20), (16385, 66000, 8), (40000, 118, 6), (300000, 17, 4), (262144, 1, 3), (100, 10, 1300), (777, 50, 2052)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_values_and_gradients(gelib, size, dtype):
    n, rows, c = size
    gen = torch.Generator(device="cuda").manual_seed(n + rows + c)
    tokens = (torch.rand(n, device="cuda", generator=gen) ** 3 * rows).long().clamp(0, rows - 1)
    tokens[torch.rand(n, device="cuda", generator=gen) < 0.1] = -1
    table = torch.randn(rows, c, device="cuda", generator=gen).to(dtype).requires_grad_()
    g = torch.randn(n, c, device="cuda", generator=gen).to(dtype)
    y = gelib.embedding(tokens, table, scale=-1.75)
    got, = torch.autograd.grad(y, table, g)
    with torch.no_grad():
        want_y, want_g, tol = reference(tokens, table.double(), g.double(), -1.75)
    check(y, want_y, u * want_y.abs(), "values of %s" % (size,))
    check(got, want_g, tol, "gradient of %s" % (size,))
    for other in (tokens, tokens.int()):   # the same bits again, from tokens of either type
        y2 = gelib.embedding(other, table, scale=-1.75)
        assert torch.equal(y2, y) and torch.equal(torch.autograd.grad(y2, table, g)[0], got)
    assert torch.equal(y, gelib.embedding(tokens, table.detach(), scale=-1.75))


def test_every_token_once_and_sorted_and_falling(gelib):
    n = 70001
    g = torch.randn(n, 12, device="cuda")
    table = torch.zeros(n, 12, device="cuda", requires_grad=True)
    for tokens in (torch.arange(n, device="cuda"), torch.arange(n - 1, -1, -1, device="cuda"), torch.randperm(n, device="cuda")):
        got, = torch.autograd.grad(gelib.embedding(tokens, table), table, g)
        assert torch.equal(got[tokens], g)


def test_runs_that_end_at_pieces(gelib):
    """Runs of one to four pieces, which begin and end at pieces' ends, one before and one behind: small whole numbers, so sums are exact."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    for lens in ([32] * 8, [64] * 6, [31, 1, 32, 33, 31], [96, 32, 64, 1, 1, 62], [1] * 100, [128] * 5, [127, 129, 128, 256, 1], [2048, 2048, 4096, 1], [1, 4095, 2048], [40000, 1, 39999]):
        tokens = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), torch.tensor(lens, device="cuda"))
        for order in (tokens, tokens[torch.randperm(len(tokens), device="cuda", generator=gen)]):
            table = torch.zeros(len(lens) + 2, 5, device="cuda", requires_grad=True)
            g = torch.randint(-8, 9, (len(order), 5), device="cuda", generator=gen).float()
            got, = torch.autograd.grad(gelib.embedding(order, table), table, g)
            assert torch.equal(got, torch.zeros_like(table).index_add(0, order, g)), lens


def test_long_sums(gelib):
    """A million terms of one sign: pieces keep chains of additions short (a chain of a million float32 additions of ones to 0.1s is
    off by 1e-3; in pieces of at most 128, three levels, 400 u = 2.4e-5)."""
    n = 1 << 20
    tokens = torch.zeros(n, device="cuda", dtype=torch.int32)
    table = torch.zeros(2, 4, device="cuda", requires_grad=True)
    g = torch.full((n, 4), 0.1, device="cuda")
    got, = torch.autograd.grad(gelib.embedding(tokens, table), table, g)
    want = float(g[0, 0].double()) * n
    assert ((got[0].double() - want).abs() <= 400 * u * want).all() and (got[1] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_tokens_outside(gelib, dtype):
    table = torch.randn(5, 24, device="cuda").to(dtype).requires_grad_()
    tokens = torch.tensor([[0, -1, 4], [5, -(1 << 62), (1 << 40) + 3]], device="cuda")
    y = gelib.embedding(tokens, table)
    assert y.shape == (2, 3, 24) and torch.equal(y[0, 0], table[0]) and (y[0, 1] == 0).all() and (y[1, 1] == 0).all()
    assert torch.isnan(y[1, 0]).all() and torch.isnan(y[1, 2]).all()
    g = torch.ones_like(y)
    g[1] = float("nan")
    got, = torch.autograd.grad(y, table, g)
    assert torch.equal(got.float(), torch.tensor([1., 0, 0, 0, 1], device="cuda")[:, None].expand(5, 24))


def test_layouts(gelib):
    table = torch.randn(40, 70, device="cuda")
    tokens = torch.randint(0, 33, (6, 50), device="cuda")
    for t in (table[:, 3:35], table.t()[:35], table[::1, ::2], table[2:36].contiguous()[:, 1:33]):
        for i in (tokens, tokens.t(), tokens[:, ::3], tokens[0, :1].expand(4, 9), tokens[0, 0], tokens[:0]):
            a, b = t.detach().requires_grad_(), t.detach().contiguous().clone().requires_grad_()
            y, z = gelib.embedding(i, a), gelib.embedding(i.contiguous(), b)
            assert y.shape == (*i.shape, t.shape[1]) and torch.equal(y, z) and torch.equal(y, t[i])
            g = torch.ones((), device="cuda").expand(y.shape)
            assert torch.equal(torch.autograd.grad(y, a, g)[0], torch.autograd.grad(z, b, g.contiguous())[0])


def test_nothing(gelib):
    table = torch.randn(0, 8, device="cuda", requires_grad=True)
    y = gelib.embedding(torch.tensor([-1, 3], device="cuda"), table)
    assert (y[0] == 0).all() and torch.isnan(y[1]).all()
    assert torch.autograd.grad(y, table, torch.ones_like(y))[0].shape == (0, 8)
    table = torch.randn(3, 8, device="cuda", requires_grad=True)
    y = gelib.embedding(torch.empty(0, 4, device="cuda", dtype=torch.int32), table)
    assert y.shape == (0, 4, 8) and (torch.autograd.grad(y, table, y)[0] == 0).all()
    y = gelib.embedding(torch.full((9,), -1, device="cuda"), table)
    assert (torch.autograd.grad(y, table, torch.ones_like(y))[0] == 0).all()


def test_against_differences_and_twice(gelib):
    """The lookup is linear: a difference is the gradient but for rounding; the gradient's gradient is a lookup."""
    tokens = torch.tensor([3, 1, 3, -1, 0], device="cuda")
    table, g, d = torch.randn(4, 6, device="cuda", requires_grad=True), torch.randn(5, 6, device="cuda", requires_grad=True), torch.randn(4, 6, device="cuda")
    y = gelib.embedding(tokens, table, scale=0.5)
    grad, = torch.autograd.grad(y, table, g, create_graph=True)
    slope = ((gelib.embedding(tokens, table + d, scale=0.5) - y).double() * g.double()).sum()
    assert abs(float(slope - (grad.double() * d).sum())) <= 1e-4
    gg, = torch.autograd.grad((grad * d).sum(), g)
    assert torch.allclose(gg, gelib.embedding(tokens, d, scale=0.5))


def test_another_stream_and_graph(gelib):
    table = torch.randn(300, 64, device="cuda").bfloat16().requires_grad_()
    tokens = torch.randint(-1, 300, (9000,), device="cuda")
    g = torch.randn(9000, 64, device="cuda").bfloat16()

    def step():
        y = gelib.embedding(tokens, table)
        return y.detach(), torch.autograd.grad(y, table, g)[0]   # (no graph outlives a step: its nodes belong to the stream that it was made on)
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
        tokens.copy_(torch.randint(-1, 300, (9000,), device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in out]
        for a, b in zip(kept, step()):
            assert torch.equal(a, b)


def test_refusals(gelib):
    table, t = torch.randn(5, 8, device="cuda"), torch.tensor([1], device="cuda")
    for bad, error in ((lambda: gelib.embedding(t.float(), table), TypeError), (lambda: gelib.embedding(t.short(), table), TypeError), (lambda: gelib.embedding(t.cpu(), table), ValueError),
                       (lambda: gelib.embedding(t, table.cpu()), ValueError), (lambda: gelib.embedding(t, table.double()), TypeError), (lambda: gelib.embedding(t, table[0]), ValueError),
                       (lambda: gelib.embedding(t, table[:, :0]), ValueError), (lambda: gelib.embedding(t, table, scale=float("nan")), ValueError)):
        with pytest.raises(error):
            bad()
