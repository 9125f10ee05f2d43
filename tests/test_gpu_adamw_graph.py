"""AdamW under graph capture: the step of one t in float32 repeats, as torch's operations would; what is rounded at random is refused, and
neither parameters nor counts have moved then."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def test_float32_replays():
    import gelib_amd as gelib
    p, q = (torch.nn.Parameter(torch.linspace(-1, 1, 900, device="cuda")) for _ in range(2))
    p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    a, b = (gelib.AdamW([t], lr=1e-2) for t in (p, q))
    for opt in (a, b):
        opt.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        b.step()
        b.set_moments(*[m.clone() for m in b.moments()], 1)   # t stays what it was when the step was recorded
        assert torch.equal(p, q)


@pytest.mark.parametrize("bits,dtype", [(8, torch.float32), (8, torch.bfloat16), (32, torch.bfloat16), (8, torch.complex64)], ids=str)
def test_rounding_at_random_is_refused(bits, dtype):
    import gelib_amd as gelib
    p = torch.nn.Parameter(torch.ones(700, device="cuda", dtype=dtype))
    p.grad = torch.ones_like(p)
    opt = gelib.AdamW([p], state_bits=bits)
    opt.step()
    torch.cuda.synchronize()
    was, kept = p.detach().clone(), [t.clone() for t in opt.moments()]
    graph, x = torch.cuda.CUDAGraph(), torch.zeros(8, device="cuda")
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="recorded"):
            opt.step()
        x += 1
    graph.replay()
    torch.cuda.synchronize()
    assert (x == 1).all() and torch.equal(p, was) and opt._groups[0].steps == [1]
    for t, k in zip(opt.moments(), kept):
        assert torch.equal(t, k)
    opt.step()
    assert not torch.equal(opt.moments()[1], kept[1]) and opt._groups[0].steps == [2]


def test_nothing_of_a_refused_step_is_recorded():
    import gelib_amd as gelib
    ps = [torch.nn.Parameter(torch.ones(300, device="cuda", dtype=t)) for t in (torch.float32, torch.bfloat16)]
    for p in ps:
        p.grad = torch.ones_like(p)
    opt = gelib.AdamW(ps)
    graph, x = torch.cuda.CUDAGraph(), torch.zeros(8, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="recorded"):
            opt.step()
        x += 1
    graph.replay()
    torch.cuda.synchronize()
    assert (x == 1).all() and all((p == 1).all() for p in ps) and opt._groups[0].steps == [0, 0]
