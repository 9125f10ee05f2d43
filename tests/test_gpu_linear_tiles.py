"""linear_act by every tile (256 x 256, 128 x 128, 64 x 128, 16 x 256) and with its sums in one, three and eight pieces, whatever the sizes
would have chosen: the comparisons of test_gpu_linear_act.py, by the same tolerances, on shapes with ragged tiles in every dimension."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests import test_gpu_linear_act as L  # noqa: E402


@pytest.fixture(scope="module")
def gelib():
    assert torch.cuda.is_available()
    import gelib_amd
    return gelib_amd


@pytest.fixture(params=[(t, s) for t in range(4) for s in (1, 3, 8)], ids=lambda p: "tile%d_pieces%d" % p)
def way(request):
    from gelib_amd import cabi
    cabi.set_option("linear_act_tile", request.param[0])
    cabi.set_option("linear_act_splits", request.param[1])
    yield request.param
    cabi.set_option("linear_act_tile", -1)
    cabi.set_option("linear_act_splits", 0)


# rows, n_in, n_out: no multiple of anything, vectors of four that end inside a tile, few steps and few rows
SHAPES = [(257, 130, 261), (300, 200, 264), (33, 520, 130), (5, 700, 40)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_values_and_gradients(gelib, way, shape, dtype):
    for act in ("none", "relu", "silu", "gelu"):
        L.test_values_and_gradients(gelib, shape, act, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gradients_are_rounded_twice_and_no_more(gelib, way, act, dtype):
    L.test_gradients_are_rounded_twice_and_no_more(gelib, act, dtype)


def test_memory_beside_the_operands_is_not_touched_or_read(gelib, way):
    L.test_memory_beside_the_operands_is_not_touched_or_read(gelib)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_layouts(gelib, way, dtype):
    L.test_layouts(gelib, dtype)


def test_infinities_stay_in_their_rows_and_columns(gelib, way):
    L.test_infinities_stay_in_their_rows_and_columns(gelib)



@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("act", ["relu", "silu", "gelu"])
def test_slopes(gelib, way, act, dtype):
    """What a tile stores of act', read back through the sum of the bias' gradient: a row of ones on one row of slopes and minus one on a
    row of slopes that are 1/2 (z = 0) leaves what differs from 1/2, which the result's type holds to a fraction of what is asked:
    2^-16 for the codes of float16 layers (steps of 2^-15 from 2^-5 on), half a step of float16 for bfloat16 layers (2^-12, from 1 on 2^-11).  The values z are those of the type,
    so that products with one are exact."""
    m, n = 300, 264
    z = torch.linspace(-3, 3, n, device="cuda").to(dtype)
    x = torch.zeros(m, 8, device="cuda", dtype=dtype)
    x[m - 1, 0] = 1   # the last row has z, the others zero
    w = torch.zeros(8, n, device="cuda", dtype=dtype)
    w[0] = z
    b = torch.zeros(n, device="cuda", dtype=dtype, requires_grad=True)
    g = torch.zeros(m, n, device="cuda", dtype=dtype)
    g[m - 1], g[0] = 1, -1
    gb, = torch.autograd.grad(gelib.linear_act(x, w, b, act=act), b, g)
    s = L.slope64(z.double(), act)
    want = s - L.slope64(torch.zeros_like(s), act)
    kept = {torch.float32: 8 * L.u, torch.bfloat16: torch.where(s >= 1, 2.0 ** -11, 2.0 ** -12), torch.float16: 2.0 ** -16}[dtype]
    assert ((gb.double() - want).abs() <= kept + 8 * L.u + L.HALF_ULP[dtype] * want.abs()).all()
