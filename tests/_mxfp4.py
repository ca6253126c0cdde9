"""MXFP4 from its definition, in 64 bits on the CPU (numpy): what the kernels are compared with."""
import numpy as np
import torch

HELD = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantise(v):
    """[..., K] numbers -> (code of every value 0..15, scale bytes [..., K / 32])."""
    v = np.asarray(v, dtype=np.float64)
    b = v.reshape(*v.shape[:-1], v.shape[-1] // 32, 32)
    largest = np.abs(b).max(-1)
    finite = np.isfinite(largest)
    safe = np.where(finite & (largest > 0), largest, 1.0)
    e = np.maximum(np.frexp(safe)[1] - 3, -127)  # floor(log2) - 2
    e = np.where(largest > 0, e, -127)
    with np.errstate(invalid="ignore", over="ignore"):
        a = np.abs(b) / np.ldexp(1.0, np.where(finite, e, 0))[..., None]
    a = np.where(finite[..., None], a, 0.0)
    middle = (HELD[1:] + HELD[:-1]) / 2
    low, high = np.searchsorted(middle, a, side="left"), np.searchsorted(middle, a, side="right")
    code = np.where((low != high) & (high % 2 == 0), high, low)  # between two codes: the even one
    code = np.where(finite[..., None], code + 8 * np.signbit(b), 0)
    scale = np.where(finite, e + 127, 255)
    return code.reshape(v.shape).astype(np.uint8), scale.astype(np.uint8)


def pack(code):
    return (code[..., 0::2] + 16 * code[..., 1::2]).astype(np.uint8)


def unpack(packed):
    return np.stack([packed & 15, packed >> 4], -1).reshape(*packed.shape[:-1], -1)


def values(code, scale):
    """What codes 0..15 and scale bytes stand for."""
    v = np.where(code >= 8, -1.0, 1.0) * HELD[code & 7]
    power = np.where(scale == 255, np.nan, np.ldexp(1.0, scale.astype(np.int64) - 127))
    return v * np.repeat(power, 32, -1)


def products(x, w, counts, row_token=None):
    """Rows [M, K] (in the order of the experts, or read through row_token) with their experts' [E, N, K]."""
    rows = len(row_token) if row_token is not None else len(x)
    out, begin = np.full((rows, w.shape[1]), np.nan), 0
    for e, n in enumerate(counts):
        at = np.arange(begin, begin + n) if row_token is None else row_token[begin:begin + n]
        there = (at >= 0) & (at < len(x))
        rows_of_e = np.where(there[:, None], x[np.where(there, at, 0)], 0.0)
        out[begin:begin + n] = rows_of_e @ w[e].T
        begin += n
    return out


def swiglu(acc, limit=0.0):
    """In 64 bits, rounded once to 32."""
    half = acc.shape[1] // 2
    g, u = acc[:, :half].astype(np.float32).astype(np.float64), acc[:, half:].astype(np.float32).astype(np.float64)
    if limit > 0:
        limit = float(np.float32(limit))
        g, u = np.minimum(g, limit), np.clip(u, -limit, limit)
    with np.errstate(over="ignore", invalid="ignore"):
        return (g / (1.0 + np.exp(-g)) * u).astype(np.float32)


def random_mx(rng, shape, spread=2, heavy=False):
    """Codes 0..15 and scales of random rows [..., K], blocks `spread` powers of two apart; heavy: large codes are rare."""
    code = rng.integers(0, 16, shape, dtype=np.uint8)
    if heavy:
        code &= rng.integers(0, 16, shape, dtype=np.uint8) | 8
    return code, (127 - 2 + rng.integers(0, spread + 1, (*shape[:-1], shape[-1] // 32))).astype(np.uint8)


def rounded(v, dtype):
    """64-bit values as a 16-bit tensor, by way of 32 bits as the kernels have them."""
    return torch.from_numpy(np.asarray(v, dtype=np.float64).astype(np.float32)).to(dtype)
