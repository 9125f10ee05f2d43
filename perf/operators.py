"""Cases of the operators around the equivariant layers: the network on invariant channels that reads vectors out
(group_norm_act, linear_act) and the training step of all weights (AdamW).

own == False computes them from elementary torch operations in 32 bits; own == True calls the framework.  Formulas:

group_norm_act(x, groups, weight, bias, eps, act, lengths), x (samples, positions, channels), a group = channels / groups
neighbouring channels over the first lengths[n] positions of sample n:
    xh = (x - mean) / sqrt(var + eps),  y = act(xh weight + bias),  zero from position lengths[n] on.
linear_act(x, w, bias, residual, act), w (n_in, n_out):  y = act(x w + bias) + residual.
AdamW, moments in 32 bits or in 8; real and imaginary parts of complex parameters are elements of their own:
    m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,
    p = p (1 - lr decay) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps).
8 bits: the elements of a tensor in blocks of 256; u = the upper 12 bits of a value's float32 pattern without sign (8 of the
exponent, 3 of the mantissa, rounded at random with random_bits below), top = the largest u of the block; a value is kept
by u - top, 254 steps of it for v (which never falls to zero from a value above zero), 126 and the sign for m (which does).
Parameters in bfloat16 are rounded at random too."""
import math
import random

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16, "complex64": torch.complex64}
EPS = 1e-5
LR, BETA1, BETA2, ADAM_EPS, DECAY, SEED, STEPS_BEFORE = 1e-4, 0.9, 0.999, 1e-8, 1e-2, 17, 100
BLOCK = 256


def norm_case(name, n, s, c, groups, dtype, act, train, ragged=False):
    return {"name": name, "op": "group_norm_act", "n": n, "s": s, "c": c, "groups": groups, "dtype": dtype, "act": act,
            "train": train, "ragged": ragged}


def linear_case(name, rows, k, n, dtype, act, residual, train):
    return {"name": name, "op": "linear_act", "rows": rows, "k": k, "n": n, "dtype": dtype, "act": act,
            "residual": residual, "train": train}


def adamw_case(name, tensors, elements, dtype, bits):
    return {"name": name, "op": "adamw", "tensors": tensors, "elements": elements, "dtype": dtype, "bits": bits}


def listed():
    return [
        # one small molecule's atoms in a served readout: a launch's latency
        norm_case("norm_serve_f32", 4, 19, 64, 8, "float32", "silu", False),
        # invariants of a batch of molecules or patches, training
        norm_case("norm_train_bf16", 64, 1024, 256, 32, "bfloat16", "silu", True),
        # the cells of the headline product (32768) one by one: as many samples as rows
        norm_case("norm_cells_f32", 32768, 1, 64, 8, "float32", "gelu", True),
        # padded grids of different sizes, ten channels a group (no power of two, no whole vector)
        norm_case("norm_ragged_bf16", 24, 9216, 320, 32, "bfloat16", "silu", True, ragged=True),
        # the readout of a single cell or token
        linear_case("linear_token_bf16", 1, 1024, 4096, "bfloat16", "silu", False, False),
        # a small batch being served, residual branch
        linear_case("linear_batch_f16", 64, 4096, 4096, "float16", "none", True, False),
        # invariants of the headline product's cells in single precision, training
        linear_case("linear_cells_f32", 32768, 256, 512, "float32", "gelu", True, True),
        # nothing a multiple of anything, rows that are not 16-byte aligned
        linear_case("linear_odd_bf16", 4099, 333, 517, "bfloat16", "silu", True, True),
        # the wide layer of a large readout
        linear_case("linear_wide_bf16", 16384, 2048, 8192, "bfloat16", "gelu", False, True),
        # the matrices of the layer behind the headline product (L = 4, 16 channels, maxl = 4): five complex matrices
        {"name": "adamw_layer_c64", "op": "adamw", "l": 4, "tau": 16, "dtype": "complex64", "bits": 32},
        # a network of many tensors, most of them small
        adamw_case("adamw_many_f32", 300, 40_000_000, "float32", 32),
        # a large one that is short of memory
        adamw_case("adamw_large_bf16_8bit", 60, 128_000_000, "bfloat16", 8),
    ]


def spread(rng, lo, hi):
    """A whole number of lo..hi, spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("group_norm_act", "linear_act", "adamw"))
    if op == "group_norm_act":
        groups, of_group = rng.choice((1, 2, 4, 8, 16, 32)), spread(rng, 1, 32)
        n = spread(rng, 1, 32768)
        s = spread(rng, 1, max(1, min(9216, 60_000_000 // (n * groups * of_group))))
        train, ragged = rng.random() < 0.6, s > 1 and rng.random() < 0.3
        # two or three values a group leave next to nothing of a gradient (none with two, but for eps): its digits are rounding
        of_group = max(of_group, 4 if ragged else -(-8 // s))
        c = norm_case("", n, s, groups * of_group, groups, rng.choice(("float32", "bfloat16", "float16")),
                      rng.choice(("none", "silu", "gelu") if train else ("none", "relu", "silu", "gelu")), train, ragged)
    elif op == "linear_act":
        rows, k = spread(rng, 1, 32768), spread(rng, 8, 4096)
        dtype = rng.choice(("float32", "bfloat16", "float16"))
        n = spread(rng, 8, max(8, min(8192, int((2e10 if dtype == "float32" else 2e11) / (rows * k)))))
        c = linear_case("", rows, k, n, dtype, rng.choice(("none", "silu", "gelu")), rng.random() < 0.5, rng.random() < 0.6)
    else:
        dtype = rng.choice(("float32", "bfloat16", "complex64"))
        elements = spread(rng, 1000, 60_000_000)
        c = adamw_case("", spread(rng, 1, max(1, min(300, elements // 500))), elements, dtype, rng.choice((8, 32)))
    del c["name"]
    return c


def tensor_sizes(case):
    """Elements of each tensor of an AdamW case (complex: of its real view)."""
    if "l" in case:
        top, tau = case["l"], case["tau"]
        pairs = [sum(abs(a - b) <= l <= a + b for a in range(top + 1) for b in range(top + 1)) for l in range(top + 1)]
        return [2 * k * tau * tau * tau for k in pairs]
    rng = random.Random(case["tensors"] * 1000003 + case["elements"])
    raw = [math.exp(rng.uniform(0.0, 5.0)) for _ in range(case["tensors"])]
    each = [max(1, int(r * case["elements"] / sum(raw))) for r in raw]
    return [n + n % 2 for n in each] if case["dtype"] == "complex64" else each


def padded(n):
    return -(-n // BLOCK) * BLOCK


def inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 2 + 1)
    dtype = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    if case["op"] == "group_norm_act":
        n, s, c = case["n"], case["s"], case["c"]
        d = {"x": randn(n, s, c).mul_(0.5 + randn(c).abs_()).add_(randn(c)).to(dtype), "w": (1 + 0.2 * randn(c)).to(dtype),
             "b": (0.2 * randn(c)).to(dtype), "lengths": None}
        if case["ragged"]:
            d["lengths"] = torch.randint(0, s + 1, (n,), device="cuda", generator=gen, dtype=torch.int32)
            d["lengths"][0] = s    # a whole sample, and behind it one with nothing in it
            d["lengths"][1:2] = 0
        if case["train"]:
            d["g"] = randn(n, s, c).to(dtype)
        return d
    if case["op"] == "linear_act":
        m, k, n = case["rows"], case["k"], case["n"]
        d = {"x": randn(m, k).to(dtype), "w": (randn(k, n) / math.sqrt(k)).to(dtype), "b": (0.2 * randn(n)).to(dtype),
             "r": randn(m, n).to(dtype) if case["residual"] else None}
        if case["train"]:
            d["g"] = randn(m, n).to(dtype)
        return d
    # parameters and gradients are slices of one buffer each, as buckets of data-parallel training have them, every one
    # from a multiple of 256 elements on; zeros in between
    sizes = tensor_sizes(case)
    total = sum(padded(k) for k in sizes)
    starts, at = [], 0
    for k in sizes:
        starts.append(at)
        at += padded(k)
    mask = torch.zeros(total, device="cuda")
    for a, k in zip(starts, sizes):
        mask[a:a + k] = 1
    flat = torch.float32 if dtype == torch.complex64 else dtype
    d = {"sizes": sizes, "starts": starts, "p": randn(total).mul_(0.05).mul_(mask).to(flat), "g": randn(total).mul_(1e-3).mul_(mask).to(flat),
         "m": randn(total).mul_(3e-4).mul_(mask), "v": randn(total).abs_().mul_(1e-6).mul_(mask)}
    if case["bits"] == 8:
        d["m"], d["v"] = as_kept(d["m"], 1 << 19, 126, False), as_kept(d["v"], 1 << 19, 254, True)
    return d


def prepare(case, seed):
    state = dict(inputs(case, seed), case=case)
    if case["op"] == "adamw":
        state["step"] = STEPS_BEFORE
        if own:
            import gelib_amd as gelib
            as_dtype = torch.view_as_complex if case["dtype"] == "complex64" else (lambda t: t)
            shaped = (lambda t: t.view(-1, 2)) if case["dtype"] == "complex64" else (lambda t: t)
            params = []
            for a, k in zip(state["starts"], state["sizes"]):
                p = torch.nn.Parameter(as_dtype(shaped(state["p"][a:a + k])))
                p.grad = as_dtype(shaped(state["g"][a:a + k]))
                params.append(p)
            state["opt"] = gelib.AdamW(params, lr=LR, betas=(BETA1, BETA2), eps=ADAM_EPS, weight_decay=DECAY, state_bits=case["bits"], seed=SEED)
            state["opt"].set_moments(state.pop("m"), state.pop("v"), STEPS_BEFORE)
    elif own and case["train"]:
        for k in ("x", "w", "b", "r"):
            if state.get(k) is not None:
                state[k].requires_grad_()
    return state


# ---- plain forms -----------------------------------------------------------------------------------------------------------

def act_of(z, act):
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return torch.clamp(z, min=0) if act == "relu" else z


def slope_of(z, act):
    if act == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return (z > 0).to(z.dtype) if act == "relu" else torch.ones_like(z)


def plain_norm(st):
    case, dtype = st["case"], st["x"].dtype
    n, s, c, k = case["n"], case["s"], case["c"], case["groups"]
    x = st["x"].float().view(n, s, k, c // k)
    w, b = st["w"].float().view(k, c // k), st["b"].float().view(k, c // k)
    if st["lengths"] is None:
        live, count = None, torch.full((n, 1, 1, 1), float(s * (c // k)), device=x.device)
    else:
        live = (torch.arange(s, device=x.device)[None, :] < st["lengths"][:, None]).view(n, s, 1, 1)
        count = (st["lengths"].float() * (c // k)).clamp(min=1).view(n, 1, 1, 1)
        x = torch.where(live, x, torch.zeros_like(x))
    mean = x.sum((1, 3), keepdim=True) / count
    d = x - mean if live is None else torch.where(live, x - mean, torch.zeros_like(x))
    rstd = torch.rsqrt((d * d).sum((1, 3), keepdim=True) / count + EPS)
    xh = d * rstd
    z = xh * w + b
    y = act_of(z, case["act"])
    y = y if live is None else torch.where(live, y, torch.zeros_like(y))
    y = y.to(dtype).view(n, s, c)
    if not case["train"]:
        return {"y": y}
    gz = st["g"].float().view(n, s, k, c // k) * slope_of(z, case["act"])
    gz = gz if live is None else torch.where(live, gz, torch.zeros_like(gz))
    gb, gw = gz.sum((0, 1)), (gz * xh).sum((0, 1))
    q = gz * w
    gx = rstd * (q - q.sum((1, 3), keepdim=True) / count - xh * ((q * xh).sum((1, 3), keepdim=True) / count))
    gx = gx if live is None else torch.where(live, gx, torch.zeros_like(gx))
    return {"y": y, "gx": gx.to(dtype).view(n, s, c), "gw": gw.to(dtype).view(c), "gb": gb.to(dtype).view(c)}


def plain_linear(st):
    case, dtype = st["case"], st["x"].dtype
    x, w = st["x"].float(), st["w"].float()
    z = torch.matmul(x, w) + st["b"].float()
    y = act_of(z, case["act"])
    y = (y if st["r"] is None else y + st["r"].float()).to(dtype)
    if not case["train"]:
        return {"y": y}
    gz = st["g"].float() * slope_of(z, case["act"])
    out = {"y": y, "gx": torch.matmul(gz, w.t()).to(dtype), "gw": torch.matmul(x.t(), gz).to(dtype), "gb": gz.sum(0).to(dtype)}
    return out if st["r"] is None else dict(out, gr=st["g"])


def random_bits(total, step, device):
    """32 random bits for every element, from its index and the step: a multiplicative mix of a counter, and 16 more."""
    a, b, c, low = 2654435769, 3144134277, 1779033703, 0xffffffff
    h = ((torch.arange(total, device=device) + (SEED * b + step * c) % 2 ** 32) * a) & low
    h = ((h ^ (h >> 15)) * b) & low
    h = ((h ^ (h >> 13)) * c) & low
    h = h ^ (h >> 16)
    h2 = (h * a) & low
    return h, (h2 ^ (h2 >> 15)) & 0xffff


def as_kept(t, add, steps, keep_above_zero):
    """The values that 8 bits keep of float32 values: add is put below the cut (random, or half for the nearest)."""
    bits = t.view(torch.int32).to(torch.int64) & 0x7fffffff
    u = ((bits + add) >> 20).view(-1, BLOCK)
    code = u - u.amax(1, keepdim=True) + steps
    kept = torch.where(code >= 1, u, u - code + 1 if keep_above_zero else torch.zeros_like(u))
    kept = torch.where(bits.view(-1, BLOCK) == 0, torch.zeros_like(u), kept)
    value = (kept << 20).to(torch.int32).view(torch.float32).view(-1)
    return torch.where(t < 0, -value, value)


def plain_adamw(st):
    st["step"] += 1
    p, g, m, v = st["p"].float(), st["g"].float(), st["m"], st["v"]
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + (g * g) * (1 - BETA2)
    denom = torch.sqrt(v) * (1 / math.sqrt(1 - BETA2 ** st["step"])) + ADAM_EPS
    p = p * (1 - LR * DECAY) - (m * (LR / (1 - BETA1 ** st["step"]))) / denom
    few = st["case"]["bits"] == 8
    if few or st["p"].dtype == torch.bfloat16:
        h, h2 = random_bits(p.numel(), st["step"], p.device)
    if few:
        m, v = as_kept(m, h & 0xfffff, 126, False), as_kept(v, h >> 12, 254, True)
    if st["p"].dtype == torch.bfloat16:
        # (a sum below 2^31 stays a number of the same sign: the values are far from the largest float)
        bits = p.view(torch.int32).to(torch.int64) & 0xffffffff
        p = ((((bits & 0x7fffffff) + h2) & ~0xffff) | (bits & 0x80000000))
        p = torch.where(p >= 1 << 31, p - (1 << 32), p).to(torch.int32).view(torch.float32)
    st["p"].copy_(p)
    st["m"].copy_(m)
    st["v"].copy_(v)
    # (a kept value has at most four significant bits: bfloat16 holds it as it is)
    return {"p": st["p"], "m": m.bfloat16() if few else st["m"], "v": v.bfloat16() if few else st["v"]}


def run(state):
    case = state["case"]
    if not own:
        return {"group_norm_act": plain_norm, "linear_act": plain_linear, "adamw": plain_adamw}[case["op"]](state)
    import gelib_amd as gelib
    if case["op"] == "adamw":
        state["opt"].step()
        m, v = state["opt"].moments()
        return {"p": state["p"], "m": m, "v": v}
    if case["op"] == "group_norm_act":
        y = gelib.group_norm_act(state["x"], case["groups"], state["w"], state["b"], eps=EPS, act=case["act"], lengths=state["lengths"])
        names = ("x", "w", "b")
    else:
        y = gelib.linear_act(state["x"], state["w"], state["b"], residual=state["r"], act=case["act"])
        names = ("x", "w", "b") if state["r"] is None else ("x", "w", "b", "r")
    if not case["train"]:
        return {"y": y}
    grads = torch.autograd.grad(y, [state[k] for k in names], state["g"])
    return dict({"g" + k: t for k, t in zip(names, grads)}, y=y.detach())


def work(case):
    e = {"float32": 4, "complex64": 4}.get(case["dtype"], 2)
    if case["op"] == "group_norm_act":
        n = case["n"] * case["s"] * case["c"]
        return {"bytes": (4 if case["train"] else 2) * e * n + 4 * e * case["c"], "flops": (40 if case["train"] else 12) * n}
    if case["op"] == "linear_act":
        m, k, n = case["rows"], case["k"], case["n"]
        values = m * k + k * n + n + m * n * (2 if case["residual"] else 1)   # x, w, b, y, r
        if case["train"]:
            values += m * n + m * k + k * n + n                               # g, gx, gw, gb
        return {"bytes": e * values, "flops": (6 if case["train"] else 2) * m * k * n}
    n = sum(tensor_sizes(case))
    moments = 16 if case["bits"] == 32 else 4 + 4                            # 8 bits: read and written, and told in 16
    return {"bytes": n * (3 * e + moments), "flops": 16 * n}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------------

def exact(case, seed):
    """From the definitions in float64, gradients by torch's differentiation of them."""
    d = inputs(case, seed)
    F = torch.nn.functional
    acts = {"none": lambda t: t, "relu": torch.relu, "silu": F.silu, "gelu": F.gelu}
    if case["op"] == "adamw":
        t = STEPS_BEFORE + 1
        p, g, m, v = (d[k].double() for k in ("p", "g", "m", "v"))
        m = torch.lerp(g, m, BETA1)
        v = torch.lerp(g.square(), v, BETA2)
        step = (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + ADAM_EPS)
        kept = case["bits"] == 32   # values rounded at random to 8 bits have no 64-bit form
        return {"p": p - LR * DECAY * p - LR * step, "m": m if kept else None, "v": v if kept else None}
    leaves = {k: d[k].double().requires_grad_(case["train"]) for k in ("x", "w", "b", "r") if d.get(k) is not None}
    if case["op"] == "linear_act":
        y = acts[case["act"]](F.linear(leaves["x"], leaves["w"].t(), leaves["b"]))
        y = y + leaves["r"] if "r" in leaves else y
    else:
        def normed(x):   # (samples, positions, channels)
            parts = x.unflatten(2, (case["groups"], -1)).transpose(1, 2).flatten(2)   # (samples, groups, positions * channels of a group)
            var, mean = torch.var_mean(parts, dim=2, correction=0, keepdim=True)
            parts = ((parts - mean) / (var + EPS).sqrt()).unflatten(2, (x.shape[1], -1)).transpose(1, 2).flatten(2)
            return acts[case["act"]](torch.addcmul(leaves["b"], parts, leaves["w"]))
        if d["lengths"] is None:
            y = normed(leaves["x"])
        else:
            if case["n"] > 4096:
                return None          # one sample at a time: minutes
            rows = []
            for k, length in enumerate(d["lengths"].tolist()):
                some = leaves["x"][k:k + 1]
                rows.append(F.pad(normed(some[:, :length]), (0, 0, 0, case["s"] - length)) if length else 0 * some)
            y = torch.cat(rows)
    if not case["train"]:
        return {"y": y}
    names = list(leaves)
    grads = torch.autograd.grad(y, [leaves[k] for k in names], d["g"].double())
    return dict({"g" + k: t for k, t in zip(names, grads)}, y=y.detach())
