"""Microscaled 4-bit matrices in numpy and float64, straight from the format's definition."""
import numpy as np

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
MIDDLE = (GRID[1:] + GRID[:-1]) / 2


def quantise(x):
    """Codes [rows][K] (0 .. 15) and scale bytes [rows][K / 32] of float64 rows."""
    b = np.asarray(x, dtype=np.float64).reshape(x.shape[0], -1, 32)
    most = np.abs(b).max(-1)
    bad = ~np.isfinite(b).all(-1)
    _, e = np.frexp(np.where(bad, 0, most) / 7)     # most / 7 = m * 2^e, m in [0.5, 1): the least e with most < 7 * 2^e
    e = np.clip(np.where(most == 0, -127, e), -127, 125)
    v = np.where(bad[..., None], 0, b) / np.exp2(e)[..., None]
    size = np.abs(v)
    below, above = np.searchsorted(MIDDLE, size, "left"), np.searchsorted(MIDDLE, size, "right")
    code = np.where(below == above, below, np.where(below % 2 == 0, below, above))
    code = code + 8 * (np.signbit(v))
    return np.where(bad[..., None], 0, code).reshape(x.shape).astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


def values(code, scale):
    """The values of codes [rows][K] and scale bytes [rows][K / 32]."""
    v = np.concatenate([GRID, -GRID])[code].reshape(code.shape[0], -1, 32)
    s = np.where(scale == 255, np.nan, np.exp2(scale.astype(np.float64) - 127))
    return (v * s[..., None]).reshape(code.shape)


def flat(code):
    """Codes two to a byte, the first in the lower four bits."""
    return (code[:, 0::2] | code[:, 1::2] << 4).astype(np.uint8)


def unflat(b):
    return np.stack([b & 15, b >> 4], -1).reshape(b.shape[0], -1)
