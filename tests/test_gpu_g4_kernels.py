"""The products of g4_kernels, which take every kernel that those of g4_reference do not, by the checks of test_gpu_g4."""
import pytest

from tests import g4_kernels as kernels
from tests import test_gpu_g4 as g4

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,N,K,group", kernels.FEW + kernels.TILES)
def test_products_of_small_integers_bit_for_bit(sess, M, N, K, group):
    g4.test_product_of_small_integers_bit_for_bit(sess, M, N, K, group)


@pytest.mark.parametrize("M,N,K,group", kernels.FEW + kernels.TILES)
def test_products_of_ordinary_rows_within_fp32_sums(sess, M, N, K, group):
    g4.test_product_of_ordinary_rows_within_fp32_sums(sess, M, N, K, group)


@pytest.mark.parametrize("M,F,K,group", kernels.FEW_SWIGLU + kernels.TILES_SWIGLU)
def test_swiglu(sess, M, F, K, group):
    g4.test_swiglu(sess, M, F, K, group)
