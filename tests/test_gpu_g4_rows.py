"""What G4 products make of a row's values: which are multiplied exactly, whatever else the row holds, and that nothing but a row's own values counts.

fp16 rows are multiplied with code - zero as they are.
"""
import numpy as np
import pytest

from rknpu2_matmul_open_amd import ops
from tests import g4_reference as ref
from tests.test_gpu_g4 import Layer, rows_of
from tests.test_gpu_mx4 import device, done, host, poisoned, ready, untouched

pytestmark = pytest.mark.gpu


class Silent(Layer):
    """Exact scales and zero points up to 15; the weights of every 37th value of K are zero, code and zero point being equal."""

    def __init__(self, sess, rng, N, K, group):
        groups = -(-K // group)
        self.where = np.arange(5 % K, K, 37)
        self.zeros = rng.integers(0, 16, (N, groups)).astype(np.uint8)
        self.code = rng.integers(0, 16, (N, K))
        self.code[:, self.where] = self.zeros[:, self.where // group]
        scales = device(rng.choice([0.5, 1.0, -1.0, 2.0], (N, groups)), "f16")
        ready()
        self.w = ops.G4Weights.from_device(sess, K, N, group, device(ref.pack(self.code)), scales, device(self.zeros))
        self.values, self.sizes = (f(self.code, host(scales), self.zeros, group) for f in (ref.weights, ref.sizes))


def run(sess, layer, x, N, K):
    ws = ops.G4Workspace(sess, x.shape[0], K, N)
    c, buf = poisoned(x.shape[0], N, "f32")
    ready()
    ws.run(layer.w, x, c)
    done(sess)
    ws.close()
    assert untouched(buf, x.shape[0], N, N)
    return host(c)


@pytest.mark.parametrize("K,group", [(1024, 128), (1024, 64), (4864, 32), (1001, 64), (999, 128)])
@pytest.mark.parametrize("M", [1, 2, 5, 9, 16, 17, 40, 100, 200])
def test_large_fp16_values_under_weights_of_zero_count_for_nothing(sess, M, K, group):
    """Beside +-61440, multiples of 2^-10 that fp32 adds exactly in any order."""
    rng = np.random.default_rng(M * 5 + K)
    N = 70
    layer = Silent(sess, rng, N, K, group)
    a = rng.integers(-4, 5, (M, K)) * 2.0 ** -10
    want = a @ layer.values.T
    assert 2.0 ** 11 * (np.abs(a) @ np.abs(layer.values).T).max() < 2 ** 24
    a[:, layer.where] = rng.choice([-61440.0, 61440.0], (M, len(layer.where)))
    got = run(sess, layer, rows_of(a, "f16"), N, K)
    assert np.array_equal(got, want), np.abs(got - want).max()
    layer.close()
