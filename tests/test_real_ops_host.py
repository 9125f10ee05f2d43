"""Operators on real channels, without a GPU: the C ABI's refusals are status codes before anything is launched, host tensors are refused,
and the random bits and 8-bit codes of AdamW are what they should be."""
import ctypes

import numpy as np
import pytest
import torch

import gelib_amd as gelib
from gelib_amd import cabi
from tests import adamw_codes as A

vp, i64, u64 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_uint64
P = vp(0x1000)


def norm(N=2, S=3, C=8, G=2, xs=24, xp=8, dtype=0, act=0, eps=1e-5, y=P, x=P, mean=None, rstd=None):
    return cabi.lib().gelib_hip_group_norm_act_fwd(y, mean, rstd, x, None, None, None, dtype, i64(N), i64(S), C, G, i64(xs), i64(xp), ctypes.c_float(eps), act, None,
                                                   u64(0), None)


def linear(rows=4, k=8, n=6, xs=8, dtype=0, act=0, y=P, x=P, w=P):
    return cabi.lib().gelib_hip_linear_act_fwd(y, None, x, w, None, None, dtype, i64(rows), k, n, i64(xs), act, None, u64(0), None)


def adamw(n=(4,), first=(0,), step=(1,), dtype=0, bits=32, lr=1e-3, b1=0.9, b2=0.99, eps=1e-8, m=P, p=P):
    k = len(n)
    A64 = i64 * k
    return cabi.lib().gelib_hip_adamw_step(k, (vp * k)(*[p] * k), (vp * k)(*[p] * k), A64(*n), A64(*first), A64(*step), m, m, None, None, dtype, bits,
                                           ctypes.c_double(lr), ctypes.c_double(b1), ctypes.c_double(b2), ctypes.c_double(eps), ctypes.c_double(0), u64(0), None)


def test_refusals_are_status_codes():
    for kw in (dict(G=3), dict(G=0), dict(C=0), dict(N=-1), dict(S=-1), dict(dtype=3), dict(dtype=-1), dict(act=4), dict(xs=-1), dict(eps=-1.0), dict(eps=float("nan")),
               dict(mean=P), dict(N=1 << 40, S=1 << 40)):
        assert norm(**kw) == 12, kw
    assert norm(y=None) == 1 and norm(x=None) == 1
    for kw in (dict(rows=-1), dict(k=-1), dict(n=-1), dict(xs=-1), dict(dtype=7), dict(act=-1), dict(rows=1 << 45)):
        assert linear(**kw) == 12, kw
    assert linear(y=None) == 1 and linear(x=None) == 1 and linear(w=None) == 1
    for kw in (dict(n=(-1,)), dict(first=(100,)), dict(first=(-256,)), dict(step=(0,)), dict(dtype=2), dict(bits=16), dict(b1=1.0), dict(b2=-0.1), dict(eps=-1.0),
               dict(lr=float("inf")), dict(n=(1 << 40,))):
        assert adamw(**kw) == 12, kw
    assert adamw(p=None) == 1 and adamw(m=None, n=(0,)) == 0 and adamw(n=(), first=(), step=()) == 0
    L = cabi.lib()
    assert L.gelib_hip_adamw_moments(P, P, P, P, P, P, i64(100), None) == 12
    assert L.gelib_hip_adamw_moments(P, P, P, P, P, None, i64(256), None) == 1
    assert L.gelib_hip_adamw_set_moments(None, P, P, P, P, P, i64(256), None) == 1
    # nothing to do is done
    assert norm(N=0, x=None, y=None) == 0 and linear(rows=0, x=None, y=None, w=None) == 0 and linear(n=0, x=None, y=None, w=None) == 0


def test_rows_of_whole_16_bytes_are_aligned():
    assert linear(k=8, xs=9) == 12 and linear(k=8, x=vp(0x1004)) == 12 and linear(n=4, w=vp(0x1008)) == 12
    # others may lie anywhere: refused only because the memory is not the device's
    assert linear(k=7, xs=9, x=vp(0x1004)) in (8, 10) and linear(k=8, rows=1, xs=9) in (8, 10)
    assert cabi.lib().gelib_hip_adamw_moments(vp(0x1008), P, P, P, P, P, i64(256), None) == 12


def test_workspaces_and_options():
    L = cabi.lib()
    assert L.gelib_hip_linear_act_workspace_bytes(0, 1, 4096, 64, 64) == 0                     # whole rows, one piece
    assert L.gelib_hip_linear_act_workspace_bytes(0, 1, 4096, 63, 64) >= 4096 * 64 * 2         # x is copied to rows of 64
    assert L.gelib_hip_linear_act_workspace_bytes(8 | 3, 1, 4096, 64, 64) >= 4096 * 64 * 2     # gz
    assert L.gelib_hip_linear_act_workspace_bytes(16, 1, 4096, 64, 64) == 0 and L.gelib_hip_linear_act_workspace_bytes(0, 5, 4096, 64, 64) == 0
    assert L.gelib_hip_group_norm_act_workspace_bytes(0, 0, 8, 3, 64, 8) == 0 and L.gelib_hip_group_norm_act_workspace_bytes(1, 0, 8, 100000, 64, 8) > 0
    for name, bad in (("linear_act_tile", 4), ("linear_act_tile", -2), ("linear_act_splits", 65), ("linear_act_other", 0)):
        with pytest.raises(cabi.GelibHipError):
            cabi.set_option(name, bad)


def test_host_memory_is_refused():
    buf = np.zeros(4096, np.float32)
    q = vp(buf.ctypes.data)
    assert norm(x=q, y=q) == 8 and linear(x=q, w=q, y=q) == 8 and adamw(p=q, m=q) == 8
    with pytest.raises(ValueError):
        gelib.group_norm_act(torch.zeros(2, 4), 2)
    with pytest.raises(ValueError):
        gelib.linear_act(torch.zeros(2, 4), torch.zeros(4, 3))
    with pytest.raises(ValueError):
        gelib.AdamW([torch.nn.Parameter(torch.zeros(2))])


def test_random_bits():
    """Every bit is set half the time and independent of its neighbours' (elements, steps, the two uses), to 5 sigma of 2^16 draws."""
    n = 1 << 16
    words = []
    for step, seed in ((1, 0), (2, 0), (1, 1), (1000003, 7 << 40)):
        h, h2 = A.random_bits(np.arange(n), step, seed)
        words.append(np.stack([(h >> b) & 1 for b in range(32)] + [(h2 >> b) & 1 for b in range(16)]).astype(np.float64) * 2 - 1)
    limit = 5 / n ** 0.5
    for w in words:
        assert np.abs(w.mean(1)).max() < limit
        own = w @ w.T / n - np.eye(len(w))
        assert np.abs(own[:32, :32]).max() < limit
        assert np.abs((w[:, :-1] * w[:, 1:]).mean(1)).max() < limit          # neighbours
    for a, b in zip(words, words[1:]):
        assert np.abs((a * b).mean(1)).max() < limit                         # steps and seeds
    far, _ = A.random_bits(np.arange(n) + (1 << 32), 1, 0)
    near, _ = A.random_bits(np.arange(n), 1, 0)
    assert (far == near).mean() < 1e-3                                       # 2^32 elements apart


def test_codes():
    rng = np.random.default_rng(1)
    x = (rng.standard_normal(2560) * np.exp(rng.uniform(-8, 0, 2560))).astype(np.float32)
    half = np.full(len(x), 1 << 19)
    y = A.kept(x, half, 126, False)
    big = np.abs(x) > np.abs(x).reshape(-1, 256).max(1).repeat(256) * 2.0 ** -15
    assert (np.abs(y - x)[big] <= np.abs(x)[big] / 16).all() and (np.abs(y - x) <= np.maximum(np.abs(x) / 16, np.abs(x).max() * 2.0 ** -15)).all()
    assert np.array_equal(A.kept(y, half, 126, False), y) and np.array_equal(A.kept(y, 0 * half + 0xfffff, 126, False), y)   # kept values stay
    v = np.abs(x) ** 2
    v[3] = 1e-30
    seen = v > v.reshape(-1, 256).max(1).repeat(256) * 2.0 ** -31   # 253 steps of an eighth of an octave below the top
    w = A.kept(v, half, 254, True)
    assert (w[v > 0] > 0).all() and (np.abs(w - v)[seen] <= v[seen] / 16).all()
    # rounding at random is right on the average
    h, _ = A.random_bits(np.arange(1 << 18), 3, 1)
    one = np.full(1 << 18, 1.03, np.float32)
    assert abs(A.kept(one, h & 0xfffff, 126, False).mean() / 1.03 - 1) < 1e-3 and abs(A.kept(one, h >> 12, 254, True).mean() / 1.03 - 1) < 1e-3
