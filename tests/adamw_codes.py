"""A host form of the AdamW step and of its 8-bit moments in numpy: float32 operations one by one, codes in integers."""
import numpy as np

LOW = 0xffffffff


def random_bits(index, step, seed):
    """(32 random bits, 16 more) of elements at these places of the moment arrays."""
    a, b, c = 2654435769, 3144134277, 1779033703
    key = (seed & LOW) * b + (seed >> 32) * a + step * c
    idx = np.asarray(index, dtype=np.uint64)
    h = ((idx & np.uint64(LOW)) + np.uint64(key & LOW) + ((idx >> np.uint64(32)) * np.uint64(b))) & np.uint64(LOW)
    h = (h * np.uint64(a)) & np.uint64(LOW)
    h = ((h ^ (h >> np.uint64(15))) * np.uint64(b)) & np.uint64(LOW)
    h = ((h ^ (h >> np.uint64(13))) * np.uint64(c)) & np.uint64(LOW)
    h = h ^ (h >> np.uint64(16))
    h2 = (h * np.uint64(a)) & np.uint64(LOW)
    return h.astype(np.int64), ((h2 ^ (h2 >> np.uint64(15))) & np.uint64(0xffff)).astype(np.int64)


def kept(x, r, steps, above_zero):
    """The values that 8 bits keep of finite float32 values of one parameter."""
    n = len(x)
    pad = -n % 256
    bits = np.pad(x.view(np.int32).astype(np.int64) & 0x7fffffff, (0, pad)).reshape(-1, 256)
    up = np.where(np.arange(n + pad).reshape(-1, 256) < n, (bits + np.pad(r, (0, pad)).reshape(-1, 256)) >> 20, 0)
    up = np.minimum(up, 2039)
    top = up.max(1, keepdims=True) if n else up[:, :1]
    code = up - top + steps
    code = np.where(code >= 1, code, 1 if above_zero else 0)
    code = np.where(bits == 0, 0, code)
    value = np.where(code == 0, 0, np.maximum(code + top - steps, 0) << 20).astype(np.int32).view(np.float32).ravel()[:n]
    return np.where(np.signbit(x), -value, value).astype(np.float32)


def to_bfloat16(x, r16):
    bits = x.astype(np.float32).view(np.uint32).astype(np.int64)
    return (((bits + r16) >> 16) << 16).astype(np.uint32).view(np.float32)


def step(p, g, m, v, lr, b1, b2, eps, decay, t):
    f = np.float32
    m = (m * f(b1) + g * f(1 - b1)).astype(f)
    v = (v * f(b2) + (g * g) * f(1 - b2)).astype(f)
    denom = (np.sqrt(v) * f(1 / np.sqrt(1 - b2 ** t)) + f(eps)).astype(f)
    return m, v, ((p - p * f(lr * decay)) - (m * f(lr / (1 - b1 ** t))) / denom).astype(f)
