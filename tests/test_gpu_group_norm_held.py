"""group_norm_act on stripes that a block holds whole in up to 16 loads a thread (8 backward), of each width of load, with ragged ends: the
same comparison with float64, by the same tolerances, as for the shapes of test_gpu_group_norm.py."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests import test_gpu_group_norm as G  # noqa: E402

# positions a thread: 16, 12 to 15, 5 to 9 of whole 16-byte loads (8 or 4 values), groups that straddle them (10 and 24 channels), several
# stripes, more samples than one; then loads of two values and of one
SHAPES = [(3, 1000, 64, 8), (2, 600, 80, 8), (3, 900, 48, 2), (2, 450, 64, 8), (3, 600, 72, 9), (2, 700, 40, 5), (3, 300, 64, 8), (5, 1024, 256, 32), (2, 1000, 10, 5),
          (3, 640, 6, 1), (2, 1100, 7, 7), (2, 560, 9, 3)]


@pytest.fixture(scope="module")
def gelib():
    assert torch.cuda.is_available()
    import gelib_amd
    return gelib_amd


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_values_and_gradients(gelib, shape, act, dtype):
    G.test_values_and_gradients(gelib, shape, act, dtype)


@pytest.mark.parametrize("shape", [(5, 1, 24, 3), (3, 40, 48, 4), (2, 900, 64, 8), (2, 30, 4100, 1)], ids=lambda s: "x".join(map(str, s)))
def test_each_gradient_by_itself(gelib, shape):
    """Whichever of x, weight and bias need a gradient, and whichever of weight and bias there are."""
    n, s, c, groups = shape
    gen = torch.Generator(device="cuda").manual_seed(6)
    x, w, b, g = (torch.randn(*k, device="cuda", generator=gen) for k in ((n, s, c), (c,), (c,), (n, s, c)))
    for given in ("xwb", "xw", "xb", "x"):
        full = {"x": x, "w": w if "w" in given else torch.ones_like(w), "b": b if "b" in given else torch.zeros_like(b)}
        leaves = {k: t.clone().requires_grad_() for k, t in full.items()}
        want = dict(zip("xwb", torch.autograd.grad(gelib.group_norm_act(leaves["x"], groups, leaves["w"], leaves["b"], act="silu"), list(leaves.values()), g)))
        for needed in ("x", "w", "b", "xw", "wb", "xb"):
            if not set(needed) <= set(given):
                continue
            ts = {k: full[k].clone().requires_grad_(k in needed) if k in given else None for k in "xwb"}
            y = gelib.group_norm_act(ts["x"], groups, ts["w"], ts["b"], act="silu")
            for k, got in zip(needed, torch.autograd.grad(y, [ts[k] for k in needed], g)):
                assert torch.equal(got, want[k]), (given, needed, k)
