"""Group-scaled 4-bit layers and the heads' norm and rotation in 64-bit numpy, from their definitions alone."""
import numpy as np

HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # of a rounding, relative to the value
LEAST = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}   # the types' smallest steps


def pack(code):
    """codes [N, K] 0..15 as bytes, the first of two in the low half."""
    code = np.pad(code, ((0, 0), (0, code.shape[1] % 2))).astype(np.uint8)
    return code[:, 0::2] | code[:, 1::2] << 4


def weights(code, scales, zeros, group):
    """w [N, K] in float64."""
    K = code.shape[1]
    wide = lambda x: np.repeat(x.astype(np.float64), group, axis=1)[:, :K]  # noqa: E731
    return (code.astype(np.float64) - (8.0 if zeros is None else wide(zeros))) * wide(scales)


def sizes(code, scales, zeros, group):
    """(code + zero) |scale|: what the terms that the kernels add are made of, at most."""
    K = code.shape[1]
    wide = lambda x: np.repeat(x.astype(np.float64), group, axis=1)[:, :K]  # noqa: E731
    return (code.astype(np.float64) + (8.0 if zeros is None else wide(zeros))) * np.abs(wide(scales))


def sum_bound(x, size, K):
    """How far sums of fp32 may be off: every term goes through up to 128 additions of its group, the scaling, the additions of all groups and those of up to 16
    waves and 16 parts, each off by 2^-23 of the terms' sum at most (2^-24 for rounding to nearest; the matrix cores need not)."""
    return (128 + K / 32 + 40) * 2.0 ** -23 * (np.abs(x) @ size.T)


def silu(g):
    with np.errstate(over="ignore"):
        return g / (1 + np.exp(-g))


def rotate(x, positions, inv_freq, pair_axis, neighbours, scale=1.0):
    """x [rows, heads, D]; positions [axes, rows]."""
    x, pairs = x.astype(np.float64), len(inv_freq)
    out = x.copy()
    for i in range(pairs):
        a, b = (2 * i, 2 * i + 1) if neighbours else (i, i + pairs)
        phi = positions[pair_axis[i]].astype(np.float64) * float(inv_freq[i])
        c, s = np.cos(phi)[:, None] * scale, np.sin(phi)[:, None] * scale
        out[:, :, a], out[:, :, b] = x[:, :, a] * c - x[:, :, b] * s, x[:, :, b] * c + x[:, :, a] * s
    return out


def head_norm(x, weight, eps):
    x = x.astype(np.float64)
    y = x / np.sqrt((x * x).mean(axis=2, keepdims=True) + eps)
    return y if weight is None else y * weight.astype(np.float64)


# Rows, columns, K and group of products: every kernel, with K in parts and not, waves that go round more than once, every number of groups in a piece, odd sizes.
SHAPES = [(1, 1, 1, 32), (1, 33, 31, 64), (1, 128, 4096, 128), (1, 70, 1001, 32), (1, 40, 9000, 64), (1, 32, 14336, 4096), (2, 64, 40, 96), (4, 200, 4360, 128),
          (4, 12300, 256, 64), (3, 1999, 2050, 50016), (5, 48, 8200, 32), (5, 12300, 520, 32), (8, 100, 8320, 128), (8, 65, 640, 320), (8, 31, 9000, 64), (9, 8200, 512, 128),
          (9, 129, 500, 64), (16, 48, 14336, 32), (16, 96, 4104, 160), (16, 8200, 1001, 64), (13, 257, 33, 32), (17, 1, 1, 32), (17, 64, 128, 128), (32, 100, 33, 64), (33, 130, 1000, 32),
          (61, 1999, 2050, 64), (64, 700, 4096, 128), (65, 257, 640, 192), (64, 96, 8192, 32), (130, 11008, 256, 64), (300, 300, 14336, 128), (33, 11800, 130, 32),
          (260, 13000, 200, 160), (200, 15490, 136, 64), (360, 5600, 280, 64), (871, 2330, 262, 128), (1370, 263, 3534, 32), (1346, 129, 2366, 128), (300, 12400, 160, 32), (1025, 6000, 384, 128), (2100, 5900, 300, 64), (77, 15000, 500, 32), (1025, 1800, 1030, 32), (129, 1000, 8192, 256)]
SWIGLU = [(1, 1, 1, 32), (1, 64, 96, 64), (1, 33, 4608, 32), (1, 40, 4360, 128), (3, 300, 4100, 64), (4, 40, 520, 160), (7, 100, 640, 32), (8, 33, 8200, 128), (16, 250, 640, 128), (16, 40, 4400, 32),
          (12, 4100, 264, 64), (17, 32, 64, 32), (31, 70, 1000, 64), (64, 500, 4096, 128), (33, 11800, 130, 32), (71, 15740, 140, 64), (300, 300, 14336, 32), (700, 3000, 264, 128), (489, 2152, 269, 128), (160, 13500, 100, 128)]
