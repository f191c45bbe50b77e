"""MX4 in 64-bit numpy, from the format's definition alone: what the tests of the MX4 operators compare with."""
import numpy as np

VALUES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)
SIGNED = np.concatenate([VALUES, -VALUES])


def quantize(x):
    """(codes uint8 [rows, 16 * blocks], scales uint8 [rows, blocks]) of x [rows, K], any float type."""
    x = np.asarray(x, np.float64)
    rows, K = x.shape
    blocks = -(-K // 32)
    v = np.zeros((rows, blocks * 32))
    v[:, :K] = x
    v = v.reshape(rows, blocks, 32)
    bad = ~np.isfinite(v).all(axis=2)
    v[bad] = 0
    most = np.abs(v).max(axis=2)
    e = np.where(most > 0, np.maximum(-127, np.frexp(most)[1] - 1 - 2), -127)
    scales = np.where(bad, 255, e + 127).astype(np.uint8)
    size = np.abs(v) / (2.0 ** e)[:, :, None]
    # the nearest value; of two equally near ones the even code
    pick, near = np.zeros(size.shape, np.uint8), np.full(size.shape, np.inf)
    for code, value in enumerate(VALUES):
        far = np.abs(size - value)
        take = (far < near) | ((far == near) & (code % 2 == 0))
        pick[take], near = code, np.minimum(far, near)
    codes = pick + 8 * np.signbit(v).astype(np.uint8)
    codes[bad] = 0
    packed = codes[:, :, 0::2] | (codes[:, :, 1::2] << 4)
    return packed.reshape(rows, blocks * 16).astype(np.uint8), scales


def values(codes, scales, K):
    """What MX4 rows stand for, float64 [rows, K]."""
    rows, blocks = scales.shape
    c = codes.reshape(rows, blocks, 16)
    both = np.stack([c & 15, c >> 4], axis=3).reshape(rows, blocks, 32)
    s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return (SIGNED[both] * s[:, :, None]).reshape(rows, blocks * 32)[:, :K]


def round_trip(x):
    return values(*quantize(x), np.asarray(x).shape[1])


def silu(g):
    return g / (1 + np.exp(-g))


def rms(x, eps, weight=None):
    y = x / np.sqrt((x * x).mean(axis=1, keepdims=True) + eps)
    return y if weight is None else y * weight


def exact_rows(rng, rows, K):
    """Random MX4 rows whose products with each other add up exactly in fp32 in any order: scales 2^0 or 2^1 -- products are multiples
    of 1/4 of at most 144, and |partial sums| of 14336 random ones stay far below 2^22.  Every block holds a 4 or a 6 (times its
    scale), so that quantizing the values gives the codes back."""
    blocks = -(-K // 32)
    code = rng.integers(0, 16, (rows, blocks, 32)).astype(np.uint8)
    code[(np.arange(blocks * 32) >= K).reshape(blocks, 32)[None].repeat(rows, 0)] = 0
    code[:, :, 0] = rng.choice([6, 7, 14, 15], (rows, blocks))
    scales = rng.choice([127, 128], (rows, blocks)).astype(np.uint8)
    packed = (code[:, :, 0::2] | (code[:, :, 1::2] << 4)).reshape(rows, blocks * 16)
    return packed, scales
