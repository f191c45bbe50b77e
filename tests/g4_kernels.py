"""Shapes of G4 products, and which kernel a product takes."""
import ctypes as C

from tests import g4_reference as ref

# Rows, columns, K and group of products that take the kernels which the shapes of g4_reference do not.
FEW = [(5, 10284, 4570, 128), (3, 30, 8654, 256), (3, 13662, 392, 128), (5, 31, 1000, 128), (9, 31, 1080, 128), (9, 30, 4192, 384),
       (9, 8193, 520, 64), (5, 10955, 4277, 192), (1, 31, 1038, 64), (2, 31, 1001, 64), (2, 31, 8376, 192), (9, 31, 1000, 64), (10, 30, 4304, 64),
       (9, 8228, 2128, 32), (1, 33, 9169, 96), (2, 30, 999, 32), (2, 30, 8293, 32), (2, 12502, 520, 96), (5, 30, 1001, 32), (9, 31, 1000, 160)]
TILES = [(2890, 663, 133, 128), (2783, 129, 5624, 256), (2467, 805, 4965, 128),
         (2142, 30, 2425, 64), (2912, 653, 654, 192), (2364, 33, 8045, 64), (1737, 3487, 137, 64), (2196, 520, 6983, 320),
         (2874, 30, 1790, 32), (2163, 1904, 2900, 96), (1532, 5339, 131, 32), (2802, 397, 5583, 160)]
FEW_SWIGLU = [(10, 4106, 520, 128), (6, 5272, 4156, 256), (1, 31, 1033, 128), (2, 31, 1001, 128), (2, 32, 4520, 256), (5, 30, 999, 128), (10, 30, 4272, 128),
              (5, 5452, 4312, 192), (1, 33, 4136, 320), (2, 31, 1000, 64), (5, 30, 1001, 64), (6, 30, 4140, 320), (10, 30, 1000, 64), (9, 32, 4216, 192),
              (9, 4090, 520, 32), (9, 4083, 2288, 160), (1, 33, 1000, 32), (2, 31, 4208, 96), (7, 30, 4136, 160), (9, 30, 1000, 32)]
TILES_SWIGLU = [(2831, 341, 133, 128), (2798, 30, 2401, 128), (2224, 65, 6938, 256), (2229, 199, 8928, 128),
                (24, 30, 1182, 64), (2846, 31, 1856, 192), (2908, 330, 652, 64), (2126, 71, 3529, 320), (2495, 1232, 131, 64), (2715, 210, 7490, 64),
                (19, 30, 924, 32), (2740, 339, 100, 32), (1880, 1087, 2651, 96), (2105, 30, 7610, 32), (2772, 1402, 136, 32), (2797, 139, 6146, 160)]


def groups_in_a_piece(group, K):
    return 1 if group >= K or group % 128 == 0 else 2 if group % 64 == 0 else 4


def _four(function, *shape):
    out = [C.c_int(0) for _ in range(4)]
    function(*shape, *map(C.byref, out))
    return [x.value for x in out]


def kernel_of(lib, M, N, K, gpb, swiglu):
    """What of the kernels' templates a product takes: few rows (rows it is made for, columns, whether waves load more than once), or tiles (rows, whether K goes in parts)."""
    kernel, rows, _, parts = _four(lib.rkh_g4_route, M, N, K, gpb, swiglu)
    if kernel:
        return ("tiles", swiglu, gpb, rows, parts > 1)
    rows, columns, _, again = _four(lib.rkh_g4_few_route, M, N, K, gpb, swiglu)
    return ("few", swiglu, gpb, rows, columns, bool(again))


def waves_of(lib, M, N, K, gpb, swiglu):
    return _four(lib.rkh_g4_few_route, M, N, K, gpb, swiglu)[2]


def taken(lib):
    """The kernels that the products of g4_reference's shapes and of these take with rows of fp16 and with rows of bf16."""
    out = set()
    for swiglu, shapes in ((0, ref.SHAPES + FEW + TILES), (1, ref.SWIGLU + FEW_SWIGLU + TILES_SWIGLU)):
        for M, N, K, group in shapes:
            if M > 16 or K % 8 == 0 or (M <= 8 <= K): # (others have rows of bf16 staged as fp16)
                out.add(kernel_of(lib, M, N, K, groups_in_a_piece(group, K), swiglu))
    return out
