"""Sums of the gradients of points over heads and pieces: with as many lanes as there are terms, up to 16.  Every number of heads, with and without
pieces (single queries of many keys), queries' points that are the keys' and that are not.  References and tolerances: test_gpu_attention.py's."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests.test_gpu_attention import compare  # noqa: E402


@pytest.fixture(scope="module")
def gelib():
    assert torch.cuda.is_available()
    import gelib_amd
    return gelib_amd


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("heads,kv", [(1, 1), (2, 1), (2, 2), (3, 1), (4, 4), (5, 5), (8, 1), (9, 3), (16, 16), (33, 11), (40, 1)])
def test_heads(gelib, heads, kv, dtype):
    compare(gelib, dtype, [(70, 70), (5, 5), (0, 0)], heads, kv, 8, False, every=False)
    compare(gelib, dtype, [(70, 90), (1, 0), (0, 5)], heads, kv, 8, True, same=False, every=False)
    compare(gelib, dtype, [(1, 900)], heads, kv, 8, False, same=False, every=False)


def test_few_rows_of_one_head(gelib):
    """Launches that end inside a block, one lane a row."""
    for n in (1, 2, 255, 256, 257, 300):
        compare(gelib, torch.float32, [(n, n)], 1, 1, 8, True, every=False)
