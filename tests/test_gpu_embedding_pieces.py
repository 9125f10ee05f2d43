"""The gradient of a table over long lists of tokens.  Sums are formed over pieces of the sorted list -- 256 entries where it has 2^18 or more, else 64 --
and what pieces share goes to lists of two entries a piece that are summed the same way.  Small whole numbers, whose float32 sums are
exact in any order: one gradient that is left out, added twice or to another row shows."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests.test_gpu_group_norm import check, u  # noqa: E402


@pytest.fixture(scope="module")
def gelib():
    assert torch.cuda.is_available()
    import gelib_amd
    return gelib_amd


# runs of one token, in order.  A piece of the second list is 64 entries, of 32 pieces of 256 tokens (8192) or of 64 (2048), of the third 32 times that
RUNS = [[255, 1, 256, 257, 255, 256, 512, 511, 513, 1, 1, 254] * 100, [256] * 1030, [8192] * 33, [8191, 1, 8192, 8193, 8191, 1] * 8, [262144], [262143, 1], [1, 262143, 2],
        [262144 - 8192, 8192, 1], [524288, 255, 1, 524288], [700001, 3, 300000], [3] * 90001, [64, 63, 65, 1, 2048, 2047, 2049, 1, 127, 129] * 20, [2048] * 120, [65536, 65535, 65537]]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("runs", RUNS, ids=lambda r: "%d of %d" % (len(r), sum(r)))
def test_runs_that_end_at_pieces(gelib, runs, dtype):
    gen = torch.Generator(device="cuda").manual_seed(len(runs))
    rows, n = len(runs), sum(runs)
    tokens = torch.repeat_interleave(torch.arange(rows, device="cuda"), torch.tensor(runs, device="cuda"))
    for channels in (1, 5, 8):
        for order in (tokens, tokens[torch.randperm(n, device="cuda", generator=gen)]):
            table = torch.zeros(rows + 2, channels, device="cuda", dtype=dtype, requires_grad=True)
            g = torch.randint(-2, 3, (n, channels), device="cuda", generator=gen)
            got, = torch.autograd.grad(gelib.embedding(order, table), table, g.to(dtype))
            want = torch.zeros(rows + 2, channels, device="cuda", dtype=torch.long).index_add_(0, order, g)
            assert torch.equal(got, want.float().to(dtype))


def test_tokens_left_out_of_long_lists(gelib):
    gen = torch.Generator(device="cuda").manual_seed(7)
    n = (1 << 18) + 777
    for rows in (1, 3, 118, 70000):
        tokens = torch.randint(-2, rows + 2, (n,), device="cuda", generator=gen)
        table = torch.zeros(rows, 4, device="cuda", requires_grad=True)
        g = torch.randint(-8, 9, (n, 4), device="cuda", generator=gen).float()
        got, = torch.autograd.grad(gelib.embedding(tokens, table), table, g)
        ok = (tokens >= 0) & (tokens < rows)
        assert torch.equal(got.double(), torch.zeros(rows, 4, device="cuda", dtype=torch.double).index_add_(0, tokens[ok], g[ok].double()))


@pytest.mark.parametrize("size", [(300000, 17, 4), (262144, 1, 3), (1 << 20, 118, 8), (40000, 118, 6)], ids=lambda s: "x".join(map(str, s)))
def test_long_random_sums(gelib, size):
    """Off by the additions that one term goes through: a piece of 256 has at most 32 single ones (what stands before and behind its whole
    sixteens), 4 levels of pairs and 16 sums of them, the lists behind it at most 32 + 4 + 4 each, of which there are three (2^20 tokens: 4096
    pieces, 8192 entries, 128 pieces, 256 entries, 4): 52 + 120 + 1 product, below 200 u of the sum of the moduli."""
    n, rows, c = size
    gen = torch.Generator(device="cuda").manual_seed(n + rows)
    tokens = (torch.rand(n, device="cuda", generator=gen) ** 3 * rows).long().clamp(0, rows - 1)
    table = torch.zeros(rows, c, device="cuda", requires_grad=True)
    g = torch.randn(n, c, device="cuda", generator=gen)
    got, = torch.autograd.grad(gelib.embedding(tokens, table), table, g)
    zero = torch.zeros(rows, c, device="cuda", dtype=torch.double)
    check(got, zero.index_add(0, tokens, g.double()), 200 * u * zero.index_add(0, tokens, g.double().abs()), "gradient of %s" % (size,))
