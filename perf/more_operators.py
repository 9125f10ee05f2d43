"""Cases of the operators of a network over points (the atoms of molecules, the cells of a grid) from its first layer to its loss:
what each point is, looked up (embedding), points of one document that look at each other (attention), a class for every point
(linear_cross_entropy), each with its gradients.

own == False computes them from elementary torch operations in 32 bits; own == True calls the framework.  Formulas:

embedding(tokens, table, scale):  y[i] = scale table[tokens[i]], a row of zeros where tokens[i] < 0;
    the gradient of row r is scale times the sum of g[i] over the i with tokens[i] == r.
attention(q, k, v, points, slopes, ...), heads h of q on heads h / (heads / kv_heads) of k and v:
    s_ij = scale q_i . k_j - slopes[h] |points_i - key_points_j|,  y_i = sum_j softmax_j(s_ij) v_j  over the keys j of i's document:
    the first lengths[n] of sample n (with query_lengths: y is zero behind them), or rows starts[d] to starts[d + 1] of packed ones;
    y_i = 0 where there are none.
linear_cross_entropy(x, w, targets, bias):  z = x w + bias,  loss[i] = log(sum_c exp z_ic) - z_i,targets[i], zero where targets[i] < 0."""
import math
import random

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def embedding_case(name, tokens, rows, channels, dtype, train, padded=0.0):
    return {"name": name, "op": "embedding", "tokens": tokens, "rows": rows, "channels": channels, "dtype": dtype, "train": train, "padded": padded}


def attention_case(name, layout, samples, queries, keys, heads, kv_heads, dim, dtype, points, train):
    """layout "padded": `samples` of `queries` and `keys` rows each, of which some exist; "packed": self-attention in `samples` documents
    of up to `keys` rows, one behind the other; "full": no mask."""
    return {"name": name, "op": "attention", "layout": layout, "samples": samples, "queries": queries, "keys": keys, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "dtype": dtype, "points": points, "train": train}


def loss_case(name, rows, k, n, dtype, train, ignored=0.0):
    return {"name": name, "op": "linear_cross_entropy", "rows": rows, "k": k, "n": n, "dtype": dtype, "train": train, "ignored": ignored}


def listed():
    return [
        # the atoms of four small molecules in a served network, by their element
        embedding_case("embed_serve_f32", 76, 118, 64, "float32", False),
        # the atoms of a large training batch: few elements, most of them the same ones, long sums
        embedding_case("embed_elements_f32", 1048576, 118, 128, "float32", True, padded=0.05),
        # a dictionary of many entries, most of which a batch does not name
        embedding_case("embed_dictionary_bf16", 65536, 65536, 2048, "bfloat16", True),
        # the same four molecules: a launch's latency
        attention_case("attn_serve_f32", "padded", 4, 19, 19, 8, 8, 8, "float32", True, False),
        # one query a sample reads a whole sample out, four heads to each head of keys
        attention_case("attn_readout_f16", "padded", 8, 1, 4099, 16, 4, 64, "float16", False, False),
        # molecules padded to the largest, single precision as the equivariant layers, forces wanted
        attention_case("attn_padded_f32", "padded", 256, 48, 48, 8, 8, 16, "float32", True, True),
        # molecules packed one behind the other, no row wasted
        attention_case("attn_packed_bf16", "packed", 2048, 60, 60, 8, 8, 32, "bfloat16", True, True),
        # a large cloud of points
        attention_case("attn_cloud_bf16", "full", 1, 8192, 8192, 16, 4, 64, "bfloat16", True, True),
        # one molecule's elements, told from what is around them
        loss_case("loss_molecule_f32", 19, 64, 118, "float32", True),
        # the elements of masked atoms: cells of the headline product (32768), 256 invariants each
        loss_case("loss_elements_f32", 32768, 256, 118, "float32", True, ignored=0.1),
        # rotations on a grid from the 455 matrix elements of l = 0..6, whose rows are not aligned
        loss_case("loss_rotations_bf16", 512, 455, 36864, "bfloat16", True),
        # the dictionary again, at the other end of the network
        loss_case("loss_dictionary_bf16", 8192, 2048, 65536, "bfloat16", True, ignored=0.1),
    ]


def spread(rng, lo, hi):
    """A whole number of lo..hi, spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("embedding", "attention", "attention", "linear_cross_entropy"))
    dtype = rng.choice(("float32", "bfloat16", "float16"))
    train = rng.random() < 0.6
    if op == "embedding":
        rows, channels = spread(rng, 1, 65536), spread(rng, 1, 2048)
        tokens = spread(rng, 1, max(1, min(1048576, 130_000_000 // channels)))
        c = embedding_case("", tokens, rows, channels, dtype, train, rng.choice((0.0, 0.2)))
    elif op == "attention":
        kv_heads, dim = spread(rng, 1, 16), rng.choice((8, 16, 32, 64, 128, spread(rng, 4, 128)))
        heads = kv_heads * rng.choice((1, 1, 2, 4, 7))
        layout = rng.choice(("padded", "packed", "full"))
        samples, points = spread(rng, 1, 1024), rng.random() < 0.6
        most = min(4e10 / dim / (4 if dtype == "float32" else 1), 1e9) / (heads * samples)   # pairs of a sample
        # (a gradient through the softmax of one or two keys is nothing but rounding)
        keys = spread(rng, 8 if train else 1, max(9, min(8192, int(math.sqrt(most)))))
        queries = rng.choice((1, keys, spread(rng, 1, keys))) if layout != "packed" else keys
        c = attention_case("", layout, samples, queries, keys, heads, kv_heads, dim, dtype, points, train)
    else:
        rows, k = spread(rng, 1, 32768), spread(rng, 8, 2048)
        n = spread(rng, 8, max(8, min(65536, int((2e10 if dtype == "float32" else 2e11) / (rows * k)))))
        c = loss_case("", rows, k, n, dtype, train, rng.choice((0.0, 0.3)))
    del c["name"]
    return c


def sizes(case):
    """The rows of each sample or document that exist: of the case, not of a seed, so that its work is known."""
    n, top = case["samples"], case["keys"]
    if case["layout"] == "full":
        return [top] * n
    rng = random.Random(n * 1000003 + top)
    few = [rng.randint((top + 7) // 8, top) for _ in range(n)]
    few[0] = top
    if n > 2:
        few[1], few[2] = 0, 1   # a document with nothing in it, one with a single row
    return few


def query_sizes(case):
    """The queries of each sample that exist: those of the keys where both are the same points, else all of them."""
    return sizes(case) if case["queries"] == case["keys"] else [case["queries"]] * case["samples"]


def inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 2 + 1)
    dtype = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    def rand(*shape):
        return torch.rand(*shape, device="cuda", generator=gen)

    def falling(n, count):
        """Numbers below n, k about 1 / (k + 1) times as often as 0: few elements and few words make up most of a text."""
        return torch.exp(rand(count).double() * math.log(n + 1)).long().sub_(1).clamp_(0, n - 1)

    if case["op"] == "embedding":
        d = {"tokens": falling(case["rows"], case["tokens"]), "table": randn(case["rows"], case["channels"]).to(dtype), "scale": 1.25}
        d["tokens"][rand(case["tokens"]) < case["padded"]] = -1
        if case["train"]:
            d["g"] = randn(case["tokens"], case["channels"]).to(dtype)
        return d
    if case["op"] == "linear_cross_entropy":
        m, k, n = case["rows"], case["k"], case["n"]
        d = {"x": randn(m, k).to(dtype), "w": (randn(k, n) * (1.5 / math.sqrt(k))).to(dtype), "b": randn(n).mul_(0.2).to(dtype), "targets": falling(n, m)}
        d["targets"][rand(m) < case["ignored"]] = -1
        if case["train"]:
            d["g"] = 0.5 + rand(m)   # a weight a row
        return d
    n, heads, kv, dim = case["samples"], case["heads"], case["kv_heads"], case["dim"]
    many = sizes(case)
    if case["layout"] == "packed":
        rows = sum(many)
        starts = [0]
        for k in many:
            starts.append(starts[-1] + k)
        # q, k and v are columns of one layer's result
        qkv = randn(rows, heads + 2 * kv, dim).to(dtype)
        q_shape, k_shape = (rows,), (rows,)
        d = {"q": qkv[:, :heads], "k": qkv[:, heads:heads + kv], "v": qkv[:, heads + kv:], "starts": torch.tensor(starts, device="cuda", dtype=torch.int32)}
    else:
        q_shape, k_shape = (n, case["queries"]), (n, case["keys"])
        d = {"q": randn(*q_shape, heads, dim).to(dtype), "k": randn(*k_shape, kv, dim).to(dtype), "v": randn(*k_shape, kv, dim).to(dtype)}
        if case["layout"] == "padded":
            d["lengths"] = torch.tensor(many, device="cuda", dtype=torch.int32)
            if case["queries"] == case["keys"]:
                d["query_lengths"] = torch.tensor(query_sizes(case), device="cuda", dtype=torch.int32)
    if case["points"]:
        side = 1.5 * max(1, case["keys"]) ** (1 / 3)   # about as dense as atoms are, in Angstrom
        d["points"] = rand(*q_shape, 3) * side
        d["key_points"] = d["points"] if case["queries"] == case["keys"] else rand(*k_shape, 3) * side
        d["slopes"] = 0.1 + rand(heads)
    if case["train"]:
        d["g"] = randn(*q_shape, heads, dim).to(dtype)
    return d


LEAVES = {"embedding": ("table",), "attention": ("q", "k", "v", "points", "key_points", "slopes"), "linear_cross_entropy": ("x", "w", "b")}


def leaves_of(state):
    """The names that gradients are asked of; points that are queries and keys are one tensor."""
    return [k for k in LEAVES[state["case"]["op"]] if state.get(k) is not None and not (k == "key_points" and state[k] is state["points"])]


def prepare(case, seed):
    state = dict(inputs(case, seed), case=case)
    if case["op"] == "attention" and case["layout"] == "packed":
        state["longest"] = max(sizes(case))
    if own and case["train"]:
        for k in leaves_of(state):
            state[k].requires_grad_()
    return state


# ---- plain forms -----------------------------------------------------------------------------------------------------------

def plain_embedding(st):
    tokens, table, scale = st["tokens"], st["table"], st["scale"]
    there = tokens >= 0
    at = torch.where(there, tokens, torch.zeros_like(tokens))
    y = torch.where(there[:, None], table[at].float() * scale, torch.zeros((), device=table.device)).to(table.dtype)
    if not st["case"]["train"]:
        return {"y": y}
    # (sums of up to a million terms: 64 bits; small tables in several copies, since adding to one place takes turns)
    copies = max(1, 65536 // len(table))
    g = torch.where(there[:, None], st["g"].double(), torch.zeros((), device=table.device, dtype=torch.float64))
    total = torch.zeros(copies * len(table), table.shape[1], device=table.device, dtype=torch.float64)
    total.index_add_(0, at + len(table) * (torch.arange(len(at), device=at.device) % copies), g)
    return {"y": y, "gtable": (total.view(copies, *table.shape).sum(0) * scale).to(table.dtype)}


def plain_attention(st):
    case, dtype = st["case"], st["q"].dtype
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    packed = case["layout"] == "packed"
    scale = 1 / math.sqrt(dim)
    if packed:   # to rows of the longest document and back
        starts, rows = st["starts"].long(), len(st["q"])
        where = starts[:-1, None] + torch.arange(st["longest"], device=starts.device)
        there = where < starts[1:, None]
        where = torch.where(there, where, torch.full_like(where, rows))

        def pad(t):
            t = torch.cat([t.float(), torch.zeros(1, *t.shape[1:], device=t.device)])
            return t[where]

        def unpad(t):
            return t[there]
        q_there = k_there = there
    else:
        pad, unpad = (lambda t: t.float()), (lambda t: t)
        lengths, q_lengths = st.get("lengths"), st.get("query_lengths")
        k_there = None if lengths is None else torch.arange(case["keys"], device=lengths.device) < lengths[:, None]
        q_there = None if q_lengths is None else torch.arange(case["queries"], device=lengths.device) < q_lengths[:, None]
    # (samples, kv heads, queries * heads of a kv head, dim): a head of keys meets all its heads of queries in one product
    q, k, v = pad(st["q"]), pad(st["k"]).transpose(1, 2), pad(st["v"]).transpose(1, 2)
    n, nq = q.shape[:2]

    def grouped(t):
        return t.unflatten(2, (kv, heads // kv)).permute(0, 2, 1, 3, 4).flatten(2, 3)

    def ungrouped(t):
        return t.unflatten(2, (nq, heads // kv)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    q = grouped(q)
    s = torch.matmul(q, k.transpose(2, 3)) * scale
    if case["points"]:
        x, p = pad(st["points"]), pad(st["key_points"])
        slope = st["slopes"].view(1, kv, 1, heads // kv, 1)
        apart = x[:, :, None, :] - p[:, None, :, :]
        dist = torch.sqrt((apart * apart).sum(3))
        s = (s.unflatten(2, (nq, -1)) - slope * dist[:, None, :, None, :]).flatten(2, 3)
    if k_there is not None:
        s = torch.where(k_there[:, None, None, :], s, torch.full((), -math.inf, device=s.device))
    top = s.amax(3, keepdim=True)
    e = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(3, keepdim=True)
    p_ = e / torch.where(total == 0, torch.ones_like(total), total)
    del s, e
    if q_there is not None:
        row = q_there.repeat_interleave(heads // kv, 1)[:, None, :, None]
        p_ = torch.where(row, p_, torch.zeros((), device=p_.device))
    y = torch.matmul(p_, v)
    out = {"y": unpad(ungrouped(y)).to(dtype)}
    if not case["train"]:
        return out
    g = grouped(pad(st["g"]))
    gv = torch.matmul(p_.transpose(2, 3), g)
    gp = torch.matmul(g, v.transpose(2, 3))
    gs = p_ * (gp - (gp * p_).sum(3, keepdim=True))
    del p_, gp
    out["gq"] = unpad(ungrouped(torch.matmul(gs, k) * scale)).to(dtype)
    out["gk"] = unpad((torch.matmul(gs.transpose(2, 3), q) * scale).transpose(1, 2)).to(dtype)
    out["gv"] = unpad(gv.transpose(1, 2)).to(dtype)
    if case["points"]:
        gs = gs.unflatten(2, (nq, -1))
        out["gslopes"] = -(gs * dist[:, None, :, None, :]).sum((0, 2, 4)).flatten()
        of_pair = -(gs * slope).sum((1, 3)) / torch.where(dist == 0, torch.ones_like(dist), dist)   # (no direction where two points are one)
        force = apart * of_pair[..., None]
        gx, gkey = force.sum(2), -force.sum(1)
        if st["key_points"] is st["points"]:
            out["gpoints"] = unpad(gx + gkey)
        else:
            out["gpoints"], out["gkey_points"] = unpad(gx), unpad(gkey)
    return out


def plain_loss(st):
    case, dtype = st["case"], st["x"].dtype
    x, w, targets = st["x"].float(), st["w"].float(), st["targets"]
    z = torch.matmul(x, w) + st["b"].float()
    there = targets >= 0
    at = torch.where(there, targets, torch.zeros_like(targets))
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    zero = torch.zeros((), device=z.device)
    loss = torch.where(there, (torch.log(total) + top - z.gather(1, at[:, None]))[:, 0], zero)
    if not case["train"]:
        return {"loss": loss}
    g = torch.where(there, st["g"], zero)
    gz = e * (g[:, None] / total)
    del z, e
    gz.scatter_add_(1, at[:, None], -g[:, None])
    return {"loss": loss, "gx": torch.matmul(gz, w.t()).to(dtype), "gw": torch.matmul(x.t(), gz).to(dtype), "gb": gz.sum(0).to(dtype)}


def run(state):
    case = state["case"]
    if not own:
        return {"embedding": plain_embedding, "attention": plain_attention, "linear_cross_entropy": plain_loss}[case["op"]](state)
    import gelib_amd as gelib
    if case["op"] == "embedding":
        y = gelib.embedding(state["tokens"], state["table"], scale=state["scale"])
    elif case["op"] == "linear_cross_entropy":
        y = gelib.linear_cross_entropy(state["x"], state["w"], state["targets"], state["b"])
    else:
        masks = {k: state.get(k) for k in ("lengths", "query_lengths", "starts")}
        y = gelib.attention(state["q"], state["k"], state["v"], state.get("points"), state.get("slopes"), key_points=state.get("key_points"), **masks)
    out = {"loss" if case["op"] == "linear_cross_entropy" else "y": y.detach()}
    if case["train"]:
        names = leaves_of(state)
        grads = torch.autograd.grad(y, [state[k] for k in names], state["g"])
        out.update({"g" + k: t for k, t in zip(names, grads)})
    return out


def work(case):
    e = {"float32": 4}.get(case["dtype"], 2)
    train = case["train"]
    if case["op"] == "embedding":
        n, c = case["tokens"], case["channels"]
        named = min(case["rows"], n)
        # forward: the rows that are named, every result; backward: every gradient, a whole table
        return {"bytes": 8 * n + e * c * (named + n) + (8 * n + e * c * (n + case["rows"]) if train else 0), "flops": n * c * (2 if train else 1)}
    if case["op"] == "linear_cross_entropy":
        m, k, n = case["rows"], case["k"], case["n"]
        values = m * k + k * n + n
        return {"bytes": e * values * (2 if train else 1) + (16 if train else 12) * m, "flops": (6 if train else 2) * m * k * n}
    rows_q, rows_k = sum(query_sizes(case)), sum(sizes(case))
    pairs = sum(a * b for a, b in zip(query_sizes(case), sizes(case)))
    values = (2 * rows_q * case["heads"] + 2 * rows_k * case["kv_heads"]) * case["dim"]                # q, y, k, v
    if train:
        values += (2 * rows_q * case["heads"] + 2 * rows_k * case["kv_heads"]) * case["dim"]           # g, gq, gk, gv
    points = (12 * (rows_q + (0 if case["queries"] == case["keys"] else rows_k)) + 4 * case["heads"]) * (2 if train else 1) if case["points"] else 0
    return {"bytes": e * values + points, "flops": pairs * case["heads"] * ((14 if train else 4) * case["dim"] + ((20 if train else 8) if case["points"] else 0))}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------------

def exact(case, seed):
    """From the definitions in float64, gradients by torch's differentiation of them."""
    d = inputs(case, seed)
    F = torch.nn.functional
    names = [k for k in LEAVES[case["op"]] if d.get(k) is not None and not (k == "key_points" and d[k] is d["points"])]
    leaf = {k: d[k].double().requires_grad_(case["train"]) for k in names}
    if case["op"] == "embedding":
        table = torch.cat([leaf["table"], leaf["table"].new_zeros(1, case["channels"])])   # a last row of zeros for what is not there
        y = F.embedding(d["tokens"] % (case["rows"] + 1), table) * d["scale"]
    elif case["op"] == "linear_cross_entropy":
        z = torch.addmm(leaf["b"], leaf["x"], leaf["w"])
        y = F.cross_entropy(z, d["targets"], ignore_index=-1, reduction="none")
    else:
        cut, packed = sizes(case), case["layout"] == "packed"

        def batch(t):
            return torch.nn.utils.rnn.pad_sequence(t.split(cut), batch_first=True) if packed else t
        q, k, v = (batch(leaf[c]).transpose(1, 2) for c in "qkv")                          # (samples, heads, rows, dim)
        k, v = (t.repeat_interleave(case["heads"] // case["kv_heads"], 1) for t in (k, v))
        if q.numel() and q.shape[2] * k.shape[2] * q.shape[0] * q.shape[1] > 1.2e9:
            return None          # (ten tensors of ten gigabytes)
        s = torch.matmul(q / math.sqrt(case["dim"]), k.transpose(2, 3))
        if case["points"]:
            x = batch(leaf["points"])
            other = batch(leaf["key_points"]) if "key_points" in leaf else x
            # (the root of the smallest number instead of zero: its slope times the zero of the square's is the zero that is meant)
            far = (x.unsqueeze(2) - other.unsqueeze(1)).square().sum(-1).clamp_min(1e-300).sqrt()
            s = s - leaf["slopes"].view(1, -1, 1, 1) * far.unsqueeze(1)
        many = torch.tensor(cut, device=s.device).view(-1, 1, 1, 1)
        s = s.masked_fill(torch.arange(s.shape[3], device=s.device) >= many, -1e300)
        y = torch.matmul(F.softmax(s, 3), v)
        live = torch.tensor(query_sizes(case), device=s.device).view(-1, 1, 1, 1) > torch.arange(s.shape[2], device=s.device).view(1, 1, -1, 1)
        y = y.masked_fill((many == 0) | live.logical_not(), 0.0).transpose(1, 2)
        if packed:
            y = torch.cat([y[n, :many] for n, many in enumerate(cut)])
    out = {"loss" if case["op"] == "linear_cross_entropy" else "y": y.detach()}
    if case["train"]:
        grads = torch.autograd.grad(y, [leaf[k] for k in names], d["g"].double())
        out.update({"g" + k: t for k, t in zip(names, grads)})
    return out
