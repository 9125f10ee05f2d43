"""The operators of a network over points together (examples/elements.py): its losses and gradients are those of torch's operations, do not change when
molecules are turned and moved, and its training runs and changes all weights."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def elements():
    assert torch.cuda.is_available()
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "elements.py")
    spec = importlib.util.spec_from_file_location("elements", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def plain(model, tokens, points, starts, targets):
    """The same network from torch's operations in 64 bits, molecule by molecule."""
    F = torch.nn.functional
    p = {k: v.double() for k, v in model.named_parameters()}
    u = p["table"][tokens]
    at = starts.tolist()
    for i in range(len(model.blocks)):
        b = {k.split(".")[-1]: v for k, v in p.items() if k.startswith("blocks.%d." % i)}
        qkv = (F.layer_norm(u, u.shape[1:], b["gain"], b["shift"]) @ b["qkv"]).view(len(u), -1, model.dim)
        q, k, v = qkv.split([model.heads, model.kv, model.kv], 1)
        k, v = (t.repeat_interleave(model.heads // model.kv, 1) for t in (k, v))
        parts = []
        for s, e in zip(at, at[1:]):
            x = points[s:e].double()
            apart = (x[:, None] - x).square().sum(2)
            far = torch.where(apart == 0, 0., torch.where(apart == 0, 1., apart).sqrt())
            z = torch.einsum("ihd,jhd->hij", q[s:e], k[s:e]) * model.dim ** -0.5 - b["slopes"][:, None, None] * far
            parts.append(torch.einsum("hij,jhd->ihd", z.softmax(2), v[s:e]))
        u = u + torch.cat(parts).flatten(1) @ b["out"]
        u = u + F.gelu(F.layer_norm(u, u.shape[1:], b["gain2"], b["shift2"]) @ b["up"]) @ b["down"]
    return F.cross_entropy(u @ p["last"] + p["bias"], targets, ignore_index=-1, reduction="none")


def test_same_as_torch(elements):
    """Float32 against 64 bits: 1e-3 of the largest gradient, some hundred roundings of 2^-24 through norms and softmaxes far from that."""
    torch.manual_seed(3)
    model = elements.Elements(elements=10, width=48, heads=6, kv_heads=2)
    tokens, points, starts, targets = elements.data(20, 10, 5)
    points.requires_grad_()
    got, want = model(tokens, points, starts, targets), plain(model, tokens, points, starts, targets)
    assert torch.allclose(got.double(), want, rtol=1e-4, atol=1e-5)
    leaves = list(model.parameters()) + [points]
    a, b = torch.autograd.grad(got.sum(), leaves), torch.autograd.grad(want.sum(), leaves)
    for p, q in zip(a, b):
        assert (p - q).abs().max() <= 1e-3 * q.abs().max() + 1e-6


def test_turned_and_moved(elements):
    torch.manual_seed(3)
    model = elements.Elements()
    tokens, points, starts, targets = elements.data(20, 16, 6)
    turn, _ = torch.linalg.qr(torch.randn(3, 3, device="cuda"))
    with torch.no_grad():
        a, b = model(tokens, points, starts, targets), model(tokens, points @ turn + 7, starts, targets)
    assert torch.allclose(a, b, rtol=1e-3, atol=1e-4)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_training(elements, dtype):
    torch.manual_seed(0)
    before = [p.detach().clone() for p in elements.Elements(dtype=dtype).parameters()]
    model, losses = elements.train(steps=6, dtype=dtype)
    assert all(torch.isfinite(p).all() for p in model.parameters()) and all(v == v for v in losses)
    assert all(not torch.equal(p, q) for p, q in zip(model.parameters(), before))
    assert elements.train(steps=3, dtype=dtype)[1] == losses[:3]   # runs repeat


def test_recorded(elements):
    """A forward and backward pass of the whole network, recorded once and replayed with other elements and places."""
    torch.manual_seed(1)
    model = elements.Elements()
    tokens, points, starts, targets = elements.data(30, 16, 7)
    leaves = list(model.parameters())

    def step():
        loss = model(tokens, points, starts, targets)
        return (loss.detach(), *torch.autograd.grad(loss.sum(), leaves))   # (no graph outlives a step: its nodes belong to the stream that it was made on)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        points.add_(0.1 * torch.randn_like(points))
        tokens.copy_(torch.randint(0, 17, tokens.shape, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in out]
        for a, b in zip(kept, step()):
            assert torch.equal(a, b)
