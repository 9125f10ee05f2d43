"""Operators of a network over points, without a GPU: the C ABI's refusals are status codes before anything is launched, host tensors are
refused, shapes without data come out right, workspaces cover what they are for."""
import ctypes

import numpy as np
import pytest
import torch

import gelib_amd as gelib
from gelib_amd import cabi

vp, i64, u64, f32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_uint64, ctypes.c_float
P = vp(0x1000)


class Desc(ctypes.Structure):
    _fields_ = [(n, vp) for n in ("q", "k", "v", "points", "key_points", "slopes", "query_marks", "key_marks")] + \
        [(n, i64) for n in ("documents", "queries", "keys")] + [(n, i64 * 3) for n in ("q_strides", "k_strides", "v_strides")] + \
        [(n, ctypes.c_int) for n in ("dtype", "packed", "heads", "kv_heads", "dim")] + [("scale", f32)]


def desc(**kw):
    d = Desc(q=0x1000, k=0x1000, v=0x1000, documents=2, queries=5, keys=5, q_strides=(i64 * 3)(160, 32, 8), k_strides=(i64 * 3)(80, 16, 8), v_strides=(i64 * 3)(80, 16, 8), heads=4,
             kv_heads=2, dim=8, scale=1.0)
    for name, v in kw.items():
        setattr(d, name, (i64 * 3)(*v) if isinstance(v, tuple) else v)
    return d


def attention(y=P, ws=None, ws_bytes=0, lse=None, **kw):
    return cabi.lib().gelib_hip_attention_fwd(ctypes.byref(desc(**kw)), y, lse, ws, u64(ws_bytes), None)


def attention_bwd(y=P, gq=P, gpoints=None, gkey=None, gslopes=None, same=0, **kw):
    return cabi.lib().gelib_hip_attention_bwd(ctypes.byref(desc(**kw)), y, P, P, gq, P, P, gpoints, gkey, gslopes, same, P, u64(1 << 40), None)


def embedding(n=4, rows=5, c=8, tb=8, dtype=0, scale=1.0, y=P, table=P, tokens=P):
    return cabi.lib().gelib_hip_embedding_fwd(y, table, tokens, tb, dtype, i64(n), i64(rows), c, f32(scale), None)


def embedding_bwd(n=4, rows=5, c=8, tb=8, dtype=0, g=P, gy=P, tokens=P, ws=P, ws_bytes=1 << 40):
    return cabi.lib().gelib_hip_embedding_bwd(g, gy, tokens, tb, dtype, i64(n), i64(rows), c, f32(1), ws, u64(ws_bytes), None)


def loss(rows=4, k=8, n=6, xs=8, dtype=0, out=P, x=P, w=P, t=P, lse=None, ws=P, ws_bytes=1 << 40):
    return cabi.lib().gelib_hip_linear_cross_entropy_fwd(out, lse, x, w, None, t, dtype, i64(rows), k, n, i64(xs), ws, u64(ws_bytes), None)


def loss_bwd(rows=4, k=8, n=6, xs=8, dtype=0, gx=P, gw=P, g=P, lse=P, t=P):
    return cabi.lib().gelib_hip_linear_cross_entropy_bwd(gx, gw, None, g, lse, P, P, None, t, dtype, i64(rows), k, n, i64(xs), P, u64(1 << 40), None)


def test_refusals_are_status_codes():
    for kw in (dict(heads=3), dict(heads=0), dict(kv_heads=0), dict(dim=0), dict(dim=129), dict(documents=-1), dict(queries=-1), dict(keys=-1), dict(dtype=3), dict(packed=2),
               dict(scale=float("nan")), dict(q_strides=(-1, 32, 8)), dict(k_strides=(80, 16, -8)), dict(v_strides=(1 << 60, 16, 8)), dict(documents=1 << 40), dict(queries=1 << 31),
               dict(keys=1 << 31), dict(points=0x1000), dict(slopes=0x1000), dict(points=0x1000, slopes=0x1000), dict(points=0x1000, key_points=0x1000)):
        assert attention(**kw) == 12, kw
        assert attention_bwd(**kw) == 12, kw
    assert attention(q=None) == 1 and attention(k=None) == 1 and attention(y=None) == 1 and attention(packed=1) == 1 and attention(packed=1, key_marks=0x1000) == 1
    assert attention(y=vp(0x1002)) == 12 and attention(q=0x1002) == 12 and attention(query_marks=0x1002) == 12
    assert attention_bwd(gpoints=P) == 12 and attention_bwd(gslopes=P) == 12   # without points there are no gradients of them
    with_points = dict(points=0x1000, key_points=0x2000, slopes=0x1000)
    assert attention_bwd(gpoints=P, same=1, **with_points) == 12 and attention_bwd(gpoints=P, same=1, queries=4, **dict(with_points, key_points=0x1000)) == 12
    assert cabi.lib().gelib_hip_attention_fwd(None, P, None, None, u64(0), None) == 1
    for kw in (dict(n=-1), dict(rows=-1), dict(rows=1 << 31), dict(c=0), dict(tb=2), dict(dtype=3), dict(n=1 << 45)):
        assert embedding(**kw) == 12 and embedding_bwd(**kw) == 12, kw
    assert embedding(scale=float("inf")) == 12 and embedding_bwd(n=1 << 31) == 12
    assert embedding(y=None) == 1 and embedding(table=None) == 1 and embedding(tokens=None) == 1 and embedding_bwd(g=None) == 1 and embedding_bwd(gy=None) == 1
    for kw in (dict(rows=-1), dict(k=-1), dict(n=0), dict(xs=-1), dict(dtype=7), dict(rows=1 << 45), dict(n=0x7fffff01)):
        assert loss(**kw) == 12 and loss_bwd(**kw) == 12, kw
    assert loss(out=None) == 1 and loss(x=None) == 1 and loss(w=None) == 1 and loss(t=None) == 1 and loss_bwd(g=None) == 1 and loss_bwd(lse=None) == 1 and loss_bwd(t=None) == 1
    assert loss(k=8, xs=9) == 12 and loss(k=8, x=vp(0x1004)) == 12 and loss(n=4, w=vp(0x1008)) == 12   # rows of whole 16 bytes are aligned
    # nothing to do is done
    assert attention(documents=0, q=None, k=None, v=None, y=None) == 0 and embedding(n=0, y=None, table=None, tokens=None) == 0 and loss(rows=0, out=None, x=None, w=None, t=None) == 0
    assert embedding_bwd(rows=0, g=None, gy=None, tokens=None) == 0


def test_workspaces():
    L = cabi.lib()
    for f in (L.gelib_hip_attention_workspace_bytes, L.gelib_hip_embedding_workspace_bytes, L.gelib_hip_linear_cross_entropy_workspace_bytes):
        f.restype = u64

    def at(what, **kw):
        return L.gelib_hip_attention_workspace_bytes(ctypes.byref(desc(**kw)), what)
    assert at(0) == 0 and at(3) == 0 and at(0, dim=129) == 0
    points = dict(points=0x1000, key_points=0x1000, slopes=0x1000)
    assert at(1) >= 2 * 5 * 4 * 4 and at(2, **points) >= at(1) + 2 * 5 * (4 + 2) * 16
    few = dict(documents=1, queries=1, keys=1 << 16, heads=1, kv_heads=1, dim=64, q_strides=(64, 64, 64), k_strides=(1 << 22, 64, 64), v_strides=(1 << 22, 64, 64))
    assert at(0, **few) >= 2 * 64 * 4     # one query's keys are cut into pieces
    assert L.gelib_hip_embedding_workspace_bytes(0, i64(1000), i64(10), 8) >= 16000 and L.gelib_hip_embedding_workspace_bytes(0, i64(0), i64(10), 8) == 0
    assert L.gelib_hip_embedding_workspace_bytes(0, i64(1000), i64(0), 8) == 0
    space = L.gelib_hip_linear_cross_entropy_workspace_bytes
    assert space(0, 1, i64(1000), 64, 100000) < 1000 * 100000 // 8                          # no logits
    assert 1 << 28 <= space(7, 1, i64(8192), 64, 1 << 20) < 1 << 30                         # some classes' gradients, not 16 GiB
    assert space(8, 1, i64(8), 8, 8) == 0 and space(0, 3, i64(8), 8, 8) == 0 and space(0, 0, i64(8), 8, 0) == 0
    # too small a workspace is refused (the memory behind it is never looked at)
    assert embedding_bwd(ws_bytes=10) in (8, 10, 13) and loss(ws=None) in (8, 10, 13)


def test_host_memory_is_refused():
    buf = np.zeros(4096, np.float32)
    q = vp(buf.ctypes.data)
    assert attention(y=q, q=q.value, k=q.value, v=q.value) == 8 and embedding(y=q, table=q, tokens=q) == 8 and loss(out=q, x=q, w=q, t=q) == 8
    with pytest.raises(ValueError):
        gelib.attention(*(torch.zeros(1, 2, 2, 4) for _ in range(3)))
    with pytest.raises(ValueError):
        gelib.embedding(torch.zeros(2, dtype=torch.long), torch.zeros(4, 3))
    with pytest.raises(ValueError):
        gelib.linear_cross_entropy(torch.zeros(2, 4), torch.zeros(4, 3), torch.zeros(2, dtype=torch.long))


def test_shapes_without_data():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        def empty(*s, dtype=torch.bfloat16):
            return torch.empty(*s, device="cuda", dtype=dtype)
        q, k, n = empty(3, 5, 4, 8), empty(3, 7, 2, 8), empty(3, dtype=torch.int32)
        x, xk, s = empty(3, 5, 3, dtype=torch.float32), empty(3, 7, 3, dtype=torch.float32), empty(4, dtype=torch.float32)
        y = gelib.attention(q, k, k, x, s, key_points=xk, lengths=n, query_lengths=n)
        assert y.shape == (3, 5, 4, 8) and y.dtype == torch.bfloat16 and y.is_cuda
        p = empty(9, 4, 8)
        assert gelib.attention(p, p, p, starts=empty(3, dtype=torch.int32)).shape == (9, 4, 8)
        y = gelib.embedding(empty(4, 5, dtype=torch.int32), empty(10, 6))
        assert y.shape == (4, 5, 6) and y.dtype == torch.bfloat16
        y = gelib.linear_cross_entropy(empty(4, 5, 8), empty(8, 9), empty(4, 5, dtype=torch.long), empty(9))
        assert y.shape == (4, 5) and y.dtype == torch.float32
        for bad in (lambda: gelib.attention(q, k, k, x, s), lambda: gelib.attention(p, p, p), lambda: gelib.embedding(empty(4, dtype=torch.int32), empty(6)),
                    lambda: gelib.linear_cross_entropy(empty(4, 8), empty(8, 9), empty(5, dtype=torch.long))):
            with pytest.raises(ValueError):
                bad()
