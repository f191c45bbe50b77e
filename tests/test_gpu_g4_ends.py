"""Rows whose K is no multiple of eight, which the few-row kernels take as they are: the last eight values are loaded together and moved to their places."""
import numpy as np
import pytest
import torch

from rknpu2_matmul_open_amd import ops
from tests import g4_reference as ref
from tests.test_gpu_g4 import Layer, row_bound, rows_of
from tests.test_gpu_mx4 import done, host, ready

pytestmark = pytest.mark.gpu

ENDS = [8297, 8298, 8299, 8300, 8301, 8302, 8303]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M", [1, 3, 5, 8])
@pytest.mark.parametrize("K", ENDS + [1004, 521, 41, 9])
def test_products_repeat_bit_for_bit(sess, M, K, group):
    """Small integers, exact in any order, and many passes: a value in a wrong place, now and then, is found."""
    rng = np.random.default_rng(M + K + group)
    N = 100
    layer = Layer(sess, rng, N, K, group)
    a = rng.integers(-4, 5, (M, K)).astype(np.float64)
    want = a @ layer.values.T
    assert 2 * (np.abs(a) @ layer.sizes.T).max() < 2 ** 24
    ws = ops.G4Workspace(sess, M, K, N)
    for kind in ("f16", "bf16"):
        x, outs = rows_of(a, kind, 3, 1), [torch.zeros((M, N), device="cuda") for _ in range(20)]
        ready()
        for c in outs:
            ws.run(layer.w, x, c)
        done(sess)
        assert all(np.array_equal(host(c), want) for c in outs), kind
    ws.close()
    layer.close()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M", [1, 3, 5, 8])
@pytest.mark.parametrize("K", [4137, 4140, 4143, 1004, 41])
def test_swiglu_repeats_and_is_within_its_bound(sess, M, K, group):
    rng = np.random.default_rng(M + K + group)
    F = 60
    layer = Layer(sess, rng, 2 * F, K, group, gate_up=True, exact=False)
    ws = ops.G4Workspace(sess, M, K, 2 * F)
    for kind in ("f16", "bf16"):
        x, outs = rows_of(rng.standard_normal((M, K)), kind), [torch.zeros((M, F), device="cuda") for _ in range(20)]
        ready()
        for c in outs:
            ws.run_swiglu(layer.w, x, c)
        done(sess)
        a = host(x)
        s, e = a @ layer.values.T, row_bound(a, layer.sizes, K)
        silu, up = ref.silu(s[:, :F]), s[:, F:]
        want = silu * up
        bound = 1.1 * e[:, :F] * (np.abs(up) + e[:, F:]) + np.abs(silu) * e[:, F:] + 2.0 ** -19 * np.abs(want) + 1e-30
        far = np.abs(host(outs[0]) - want) - bound - ref.HALF_STEP["f32"] * (np.abs(want) + bound)
        assert far.max() <= 0, (kind, far.max())
        assert all(torch.equal(c, outs[0]) for c in outs), kind
    ws.close()
    layer.close()
