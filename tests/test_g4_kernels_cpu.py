"""Every kernel that a G4 product can take is one that a test takes: by what the dispatch decides, which is arithmetic."""
import numpy as np
import pytest

from rknpu2_matmul_open_amd import capi
from tests import g4_kernels as kernels


@pytest.fixture(scope="module")
def lib():
    return capi.load_library()


def products(n, seed):
    rng = np.random.default_rng(seed)
    log = lambda lo, hi: int(np.exp(rng.uniform(np.log(lo), np.log(hi))))  # noqa: E731
    for i in range(n):
        M = log(1, 17) if i % 2 else log(17, 3000)
        yield M, log(1, 40000), log(1, 40000), int(rng.choice([1, 2, 4])), i // 2 % 2


def test_every_kernel_is_taken_by_a_tested_product(lib):
    tested, reached = kernels.taken(lib), set()
    for M, N, K, gpb, swiglu in products(120000, 1):
        reached.add(kernels.kernel_of(lib, M, N, K, gpb, swiglu))
    # all tiles with and without parts; few rows: operands, 1, 4, 8 and 16 rows, each loading once or more, and 4 rows x 32 columns for results that are no pairs
    assert reached == {("tiles", s, g, rows, parts) for s in (0, 1) for g in (1, 2, 4) for rows in (32, 64, 128, 256) for parts in (False, True)} | {
        ("few", s, g, rows, 64 if rows == 0 else 32 if s else 16, again) for s in (0, 1) for g in (1, 2, 4) for rows in (0, 1, 4, 8, 16) for again in (False, True)} | {
        ("few", 0, g, 4, 32, False) for g in (1, 2, 4)}
    assert reached <= tested, sorted(reached - tested)


def test_waves_of_few_rows_fit_their_kernels(lib):
    """A workgroup has no more waves than its kernel is bounded by (eight where registers are many), all of which have work."""
    for M, N, K, gpb, swiglu in products(60000, 2):
        kind = kernels.kernel_of(lib, M, N, K, gpb, swiglu)
        if kind[0] != "few":
            continue
        _, _, _, rows, columns, _ = kind
        waves, pieces = kernels.waves_of(lib, M, N, K, gpb, swiglu), -(-K // 128)
        most = 8 if rows == 16 or (swiglu and rows) or (rows == 4 and columns == 32) or (gpb == 4 and rows in (0, 8)) else 16
        assert 1 <= waves <= min(most, pieces), (M, N, K, gpb, swiglu, waves)
        assert rows == 0 or M <= rows
