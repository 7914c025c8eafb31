"""64-bit restatement of the 8-bit activation form and of the operators that use it, for the tests."""
import numpy as np

BLOCK = 32
E4M3 = np.array([(-1.0) ** (b >> 7) * (2.0 ** ((b >> 3 & 15) - 7) * (1 + (b & 7) / 8) if b >> 3 & 15 else (b & 7) * 2.0 ** -9) for b in range(256)])
E4M3[[0x7F, 0xFF]] = np.nan


def bf16(x):
    """To the nearest BF16 (ties to even), as float64; NaN stays NaN, overflow is infinite."""
    import torch
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float64)).to(torch.bfloat16).double().numpy()


def blocks(v):
    rows, D = v.shape
    n = -(-D // BLOCK)
    full = np.zeros((rows, n * BLOCK))
    full[:, :D] = v
    return full.reshape(rows, n, BLOCK)


def exponent(amax):
    """The smallest whole k with amax <= 448 * 2^k, in [-117, 119]; -117 for 0."""
    with np.errstate(divide="ignore"):
        m, e = np.frexp(amax)
    return np.where(amax == 0, -117, np.clip(np.where(m > 0.875, e - 8, e - 9), -117, 119)).astype(np.int64)


def pack(v):
    """float64 [rows, D] -> (bytes of e4m3, scale bytes)."""
    rows, D = v.shape
    b = blocks(v)
    finite = np.isfinite(b)
    k = exponent(np.abs(np.where(finite, b, 0.0)).max(-1))
    x = np.where(finite, b, np.nan) * np.exp2(-k.astype(np.float64))[..., None]
    mag = np.minimum(np.abs(x), 448.0)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.maximum(np.frexp(mag)[1] - 1, -6)
        steps = np.rint(np.ldexp(mag, 3 - e))              # half to even
    steps = np.where(np.isnan(steps), 0, steps).astype(np.int64)
    up = steps == 16                                       # rounded up into the next binade
    e, steps = np.where(up, e + 1, e), np.where(up, 8, steps)
    code = np.where(steps >= 8, ((e + 7) << 3) + (steps - 8), steps)
    code = np.where(np.isnan(x), 0x7F, code | (np.signbit(x).astype(np.int64) << 7))
    return code.reshape(rows, -1)[:, :D].astype(np.uint8), (k + 127).astype(np.uint8)


def widen(q, scale):
    D = q.shape[1]
    return E4M3[q] * np.exp2(scale.astype(np.float64) - 127).repeat(BLOCK, axis=1)[:, :D]


def activations(rng, rows, D, size=1.0):
    """BF16-valued rows: tokens of unlike size, a few channels far above the rest, some rows of zeros."""
    x = rng.standard_normal((rows, D)) * np.exp(0.5 * rng.standard_normal((rows, 1))) * size
    x[:, rng.integers(0, D, max(1, D // 256))] *= 24.0
    x[rng.random(rows) < 0.05] = 0.0
    return bf16(x)


def sigmoid(x):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-x))
