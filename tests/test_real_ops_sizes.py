"""The operators on real channels at sizes where 32-bit indexes and the limits of a launch end.  Rows and columns that are compared
are few; everything else is there to be counted past."""
import ctypes

import pytest
import torch

import gelib_amd as gelib
from gelib_amd import cabi

i64 = ctypes.c_int64


@pytest.fixture(autouse=True)
def memory():
    yield
    if torch.cuda.is_available():
        torch.cuda.empty_cache()


def scribbled(sizes):
    """Memory of these sizes that the next allocations get holds sixes: what is not written does not pass for a result."""
    torch.cuda.empty_cache()
    ts = [torch.full((n,), 0x66, device="cuda", dtype=torch.uint8) for n in sizes]
    del ts


def linear_workspace(what, dtype, rows, k, n):
    return cabi.lib().gelib_hip_linear_act_workspace_bytes(what, dtype, i64(rows), k, n)


def test_a_few_rows_of_many_columns_go_to_the_tiles():
    """Without a workspace: one launch without tiles.  A row of one value is copied to 16 bytes for the tiles."""
    assert linear_workspace(0, 1, 4, 1, 1 << 27) == 0
    for n in (1 << 28, 800000000, 2000000000):
        assert linear_workspace(0, 1, 4, 1, n) > 0


def test_workspaces_of_wide_odd_rows():
    """Copies to rows of whole 16 bytes, of 2^31 bytes and more each: the size that is asked for is theirs and what pieces may add."""
    for dtype, e, n in ((1, 2, (1 << 30) + 1), (0, 4, (1 << 29) + 1), (2, 2, (1 << 31) - 1025)):
        copy = -(-n * e // 16) * 16
        assert 0 <= linear_workspace(0, dtype, 5, 8, n) - 8 * copy <= 1024               # w
        assert 0 <= linear_workspace(0, dtype, 5, n, 8) - 5 * copy <= 64 * 8 * 5 * 4 + 1024   # x, 64 pieces
        assert 0 <= linear_workspace(8 | 2, dtype, 3, 8, n) - 3 * copy <= 1024           # gz


def test_widths_that_do_not_round_up_within_31_bits():
    """Widths are rounded up to vectors and tiles: within 255 of 2^31 they are refused, by either side, before anything else is looked at."""
    L, vp = cabi.lib(), ctypes.c_void_p
    most = (1 << 31) - 256
    for k, n in ((most, 1), (1, most), (most + 1, 1), (1, most + 1), ((1 << 31) - 1, 8), (8, (1 << 31) - 1)):
        args = (1, i64(2), k, n, i64(k))
        fwd = L.gelib_hip_linear_act_fwd(None, None, None, None, None, None, *args, 0, None, 0, None)
        bwd = L.gelib_hip_linear_act_bwd(None, None, None, None, None, None, None, *args, None, 0, None)
        assert (fwd, bwd) == ((1, 1) if max(k, n) <= most else (12, 12))
        assert (linear_workspace(2, 1, 2, k, n) == 0) == (max(k, n) > most)


@pytest.fixture
def two_pieces():
    cabi.set_option("linear_act_tile", 3)
    cabi.set_option("linear_act_splits", 2)
    yield
    cabi.set_option("linear_act_tile", -1)
    cabi.set_option("linear_act_splits", 0)


MANY_ROWS = (1 << 26) + 100   # more than 2^22 tiles of 16 rows: two launches


def test_products_of_several_launches_are_not_cut_into_pieces(two_pieces):
    assert linear_workspace(0, 1, 1000, 72, 8) >= 2 * 1000 * 8 * 4
    assert linear_workspace(0, 1, MANY_ROWS, 72, 8) == 0


@pytest.mark.gpu
def test_rows_of_several_launches(two_pieces):
    x = torch.zeros(MANY_ROWS, 72, device="cuda", dtype=torch.bfloat16)
    x[:200].normal_()
    x[-200:].normal_()
    w = torch.randn(72, 8, device="cuda").bfloat16()
    y = gelib.linear_act(x, w)
    for part in (slice(0, 200), slice(-200, None)):
        want = x[part].double() @ w.double()
        assert ((y[part].double() - want).abs() <= 2.0 ** -8 * want.abs() + 80 * 2.0 ** -24 * (x[part].double().abs() @ w.double().abs())).all()
    assert not y[200:-200].any()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1 << 27, (1 << 28) + 8, 800000000])
def test_a_few_rows_of_many_columns(n):
    """The last row's last result lies behind 2^31 elements at 800 million columns (y: 6.4 GB)."""
    x = torch.tensor([[1.0], [-2.0], [3.0], [0.5]], device="cuda", dtype=torch.bfloat16)
    w = torch.ones(1, n, device="cuda", dtype=torch.bfloat16)
    w[0, -3:] = torch.tensor([4.0, 5.0, 6.0])
    y = gelib.linear_act(x, w)
    assert y.shape == (4, n)
    for m in range(4):
        assert (y[m, :-3] == x[m]).all() and torch.equal(y[m, -3:], x[m] * w[0, -3:])


@pytest.mark.gpu
@pytest.mark.parametrize("n", [(1 << 29) + 8, (1 << 30) + 1])
def test_column_sums_of_many_columns(n):
    """One row, so every sum is one value; behind 2^30 columns of an odd number also the copy of the gradient to aligned rows."""
    x = torch.full((1, 1), 2.0, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w = torch.zeros(1, n, device="cuda", dtype=torch.bfloat16)
    w[0, -4:] = torch.tensor([1.0, 2.0, 3.0, 4.0])
    w.requires_grad_()
    b = torch.zeros(n, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    g = torch.ones(1, n, device="cuda", dtype=torch.bfloat16)
    g[0, ::1000003] = 5.0
    g[0, -1] = 7.0
    y = gelib.linear_act(x, w, b)
    scribbled(3 * [2 * n] + [4 * n])
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), g)
    assert torch.equal(gb, g[0]) and torch.equal(gw, 2 * g)
    assert gx.item() == (g[0, -4:] * w[0, -4:]).sum().item()


@pytest.mark.gpu
@pytest.mark.parametrize("n,s,c,groups", [((1 << 22) + 8, 1, 1031, 1), ((1 << 20) + 16, 241, 65, 65)])
def test_norms_of_many_groups(n, s, c, groups):
    """More groups than one launch has blocks (1024 threads a group of many pieces) or waves for: the last samples are what they are by
    themselves, but for the order of sums."""
    x = torch.zeros(n, s, c, device="cuda", dtype=torch.bfloat16)
    for part in (x[:3], x[-9:]):
        part.normal_()
    scribbled([cabi.lib().gelib_hip_group_norm_act_workspace_bytes(0, 1, i64(n), i64(s), c, groups), x.numel() * 2])
    y = gelib.group_norm_act(x, groups)
    for part in (slice(0, 3), slice(-9, None)):
        alone = gelib.group_norm_act(x[part].contiguous(), groups)
        assert ((y[part].float() - alone.float()).abs() <= 2.0 ** -7 * alone.float().abs() + 1e-4).all()
    assert not y[3:-9].any()


@pytest.mark.gpu
def test_norms_of_many_stripes():
    """16777217 channels in groups of 97 are 86481 stripes of two groups."""
    from tests.test_gpu_group_norm import check, reference
    c, groups = 16777217, 172961
    gen = torch.Generator(device="cuda").manual_seed(1)
    x, w, b, g = (torch.randn(*k, device="cuda", generator=gen) for k in ((1, 1, c), (c,), (c,), (1, 1, c)))
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = gelib.group_norm_act(x, groups, w, b, act="silu")
    got = dict(zip(("gx", "gw", "gb"), torch.autograd.grad(y, leaves, g)), y=y.detach())
    with torch.no_grad():
        want = reference(x.double(), groups, w.double(), b.double(), 1e-5, "silu", torch.ones(1, device="cuda", dtype=torch.long), g.double())
    for k, t in got.items():
        check(t, want[k][0].reshape(t.shape), want[k][1].reshape(t.shape), k)


@pytest.mark.gpu
def test_norms_of_many_chunks():
    """67 million positions of 129 channels in chunks of 16: more than a launch takes.  Zeros but for both ends, so that the formulas are
    sums over these; a value is rounded to bfloat16 and the statistics to far less."""
    s, c = (1 << 26) + 33, 129
    ends = [slice(0, 40), slice(-40, None)]
    x, g = (torch.zeros(1, s, c, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    for t in (x, g):
        for e in ends:
            t[0, e].normal_()
    leaf = x.requires_grad_()
    y = gelib.group_norm_act(leaf, 1, eps=1e-3)
    gx, = torch.autograd.grad(y, leaf, g)
    X, G = (torch.cat([t.detach()[0, e].double() for e in ends]) for t in (x, g))
    mean = X.sum() / (s * c)
    rstd = ((X.square().sum()) / (s * c) - mean.square() + 1e-3).rsqrt()
    xh = (X - mean) * rstd
    want_y, want_gx = xh, rstd * (G - G.sum() / (s * c) - xh * ((G * xh).sum() / (s * c)))
    for got, want in ((y, want_y), (gx, want_gx)):
        mine = torch.cat([got.detach()[0, e].double() for e in ends])
        assert ((mine - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -12 * want.abs().max()).all()
        assert got.detach()[0, 40:-40].abs().max() <= 1e-2


@pytest.mark.gpu
def test_gradients_with_a_graph_of_groups_of_2_31_values():
    """The gradients that have a graph (torch's operations) are those of the kernels."""
    s, c = 131073, 16384
    gen = torch.Generator(device="cuda").manual_seed(2)
    x, g = (torch.randn(1, s, c, device="cuda", generator=gen, dtype=torch.bfloat16) for _ in range(2))
    lengths = torch.full((1,), s, device="cuda", dtype=torch.int32)
    leaf = (x + 3).requires_grad_()
    y = gelib.group_norm_act(leaf, 1, lengths=lengths)
    a, = torch.autograd.grad(y, leaf, g, retain_graph=True)
    b, = torch.autograd.grad(y, leaf, g, create_graph=True)
    b = b.detach()
    for part in (slice(0, 500), slice(-500, None)):
        assert ((a[0, part].float() - b[0, part].float()).abs() <= 2.0 ** -7 * a[0, part].float().abs() + 1e-4).all()
