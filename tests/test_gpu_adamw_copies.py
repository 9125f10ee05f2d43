"""Copies of an AdamW optimizer, by copy.deepcopy and by pickle: they hold parameters and moments of their own and go on as the original does."""
import copy
import io
import pickle

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def made(bits):
    import gelib_amd as gelib
    gen = torch.Generator(device="cuda").manual_seed(3)
    model = torch.nn.ParameterList([torch.nn.Parameter(torch.randn(*n, device="cuda", generator=gen)) for n in ((300,), (20, 30), (7,))])
    model.append(torch.nn.Parameter(torch.randn(5, 6, device="cuda", generator=gen).bfloat16()))
    model.append(torch.nn.Parameter(torch.randn(5, 6, device="cuda", generator=gen, dtype=torch.complex64)))
    ps = list(model)
    return model, gelib.AdamW([{"params": ps[:2]}, {"params": ps[2:], "lr": 0.1, "weight_decay": 0.0}], lr=1e-2, state_bits=bits, seed=5)


def step(model, opt, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    for k, p in enumerate(model):
        p.grad = torch.randn(p.shape, device="cuda", generator=gen, dtype=p.dtype) if k != 1 or seed != 1 else None   # one is left out once
    opt.step()


def by_pickle(pair):
    buf = io.BytesIO()
    pickle.dump(pair, buf)
    buf.seek(0)
    return pickle.load(buf)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("how", [copy.deepcopy, by_pickle])
def test_a_copy_goes_on(how, bits):
    model, opt = made(bits)
    for seed in (0, 1):
        step(model, opt, seed)
    other, twin = how((model, opt))
    assert all(a is not b for a, b in zip(other, model)) and all(a is b for a, b in zip(other, [p for g in twin.param_groups for p in g["params"]]))
    assert [list(g.steps) for g in twin._groups] == [list(g.steps) for g in opt._groups] == [[2, 1], [2, 2, 2]]
    was = [p.detach().clone() for p in model]
    step(other, twin, 2)
    assert all(torch.equal(p, q) for p, q in zip(model, was))          # the original's are its own
    step(model, opt, 2)
    for p, q in zip(model, other):
        assert torch.equal(p, q)
        for a, b in zip(opt.moments(p), twin.moments(q)):
            assert torch.equal(a, b)
    # and the copy's state loads into the original, a further group finds its place in the copy
    opt.load_state_dict(twin.state_dict())
    late = torch.nn.Parameter(torch.zeros(400, device="cuda"))
    twin.add_param_group({"params": [late], "lr": 0.5, "weight_decay": 0.0})
    late.grad = torch.ones_like(late)
    step(other, twin, 3)
    step(model, opt, 3)
    assert all(torch.equal(p, q) for p, q in zip(model, other)) and ((late.detach() + 0.5).abs() < 1e-5).all()
