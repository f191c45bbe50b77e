"""What G4 products make of a row's values: which are multiplied exactly, whatever else the row holds, and that nothing but a row's own values counts.

fp16 rows are multiplied with code - zero as they are.  bf16 rows of up to 16 are multiplied with the code, and zero times the group's sum is taken off; more of them are
staged as halves: exact down to 2^-31 of the row's largest value (that is moved to 2^14 .. 2^15, and the eight bits of a value of 2^-17 end at 2^-24, a half's smallest step),
off by half of a step, 2^-39 of the largest value's power of two, below.
"""
import numpy as np
import pytest
import torch

from rknpu2_matmul_open_amd import ops
from tests import g4_reference as ref
from tests.test_gpu_g4 import Layer, row_bound, rows_of
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


@pytest.mark.parametrize("K", [1024, 264, 999])
@pytest.mark.parametrize("M", [17, 40, 100, 200])
def test_staged_bf16_rows_are_exact_down_to_2_31_of_their_largest_value(sess, M, K):
    """The largest value counts for nothing; the others are 128 .. 255 times 2^-38 of its power of two, which fp32 adds exactly in any order, and then of 2^-39 .. 2^-48."""
    rng = np.random.default_rng(M + K)
    N = 70
    layer = Silent(sess, rng, N, K, 64)
    assert 2.0 * 255 * np.abs(layer.values).sum(1).max() < 2 ** 24
    for largest, below in ((1.0, 38), (1.9921875, 38), (1.0, 39), (1.9921875, 39), (1.5, 41), (1.0, 44), (1.0, 48)):
        power = np.exp2(rng.integers(-60, 100, (M, 1)))
        a = rng.integers(128, 256, (M, K)) * rng.choice([-1.0, 1.0], (M, K)) * 2.0 ** -below * power
        a[:, layer.where] = 0.0
        want = a @ layer.values.T
        a[:, layer.where] = largest * power * rng.choice([-1.0, 1.0], (M, len(layer.where)))
        got = run(sess, layer, rows_of(a, "bf16"), N, K)
        if below == 38:
            assert np.array_equal(got, want), (largest, np.abs(got / want - 1).max())
        else: # (halves of 2^-25 and its multiples: sums of them are exact as well)
            far = np.abs(got - want) - 2.0 ** -39 * power * np.abs(layer.values).sum(1)
            assert far.max() <= 0, (largest, below)
    layer.close()


@pytest.mark.parametrize("M", [1, 4, 8, 16, 17, 40, 200])
def test_bf16_sums_are_finite_up_to_2_113(sess, M):
    """A group of 128 values below 2^113 of one sign under zero points of 255: its sums stay below 2^128, in either form."""
    rng = np.random.default_rng(M)
    N, K, group = 70, 640, 128
    code, zeros = rng.integers(0, 16, (N, K)), np.full((N, K // group), 255, np.uint8)
    scales = np.exp2(rng.integers(-9, -5, (N, K // group)))
    w = ops.G4Weights(sess, K, N, group, ref.pack(code), scales.astype(np.float16), zeros)
    values, sizes = (f(code, scales, zeros, group) for f in (ref.weights, ref.sizes))

    class Holder:
        pass
    layer = Holder()
    layer.w = w
    a = rng.integers(128, 256, (M, K)) * 2.0 ** 105 * rng.choice([-1.0, 1.0], (M, 1))
    got, want = run(sess, layer, rows_of(a, "bf16"), N, K), a @ values.T
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= row_bound(a, sizes, K) + ref.HALF_STEP["f32"] * np.abs(want)).all()
    w.close()


SHAPES = [(1, 200, 4096, 128), (8, 200, 4096, 32), (8, 4096, 14336, 128), (16, 12300, 640, 64), (40, 700, 4096, 64), (64, 96, 8192, 32), (100, 300, 1001, 128), (300, 300, 14336, 128),
          (300, 6000, 520, 32)]


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("M,N,K,group", SHAPES)
def test_rows_keep_their_bits_beside_any_others_and_from_call_to_call(sess, M, N, K, group, kind):
    """A third of the rows stays; the others are replaced by rows of other sizes, with infinities and NaN among them.  The first rows are multiplied again at the end."""
    rng = np.random.default_rng(M + N)
    layer = Layer(sess, rng, N, K, group, exact=False)
    kept = np.arange(M) % 3 == 0
    a = rng.standard_normal((M, K)) * np.exp2(rng.integers(-6, 3, (M, 1)))
    first = run(sess, layer, rows_of(a, kind), N, K)
    assert np.isfinite(first).all()
    for turn in range(3):
        b = rng.standard_normal((M, K)) * np.exp2(rng.integers(-12, 9, (M, 1)))
        b[:, rng.integers(0, K, 8)] *= 50
        b[kept] = a[kept]
        x = rows_of(b, kind)
        for r in np.flatnonzero(~kept)[turn::4]:
            x[r, int(rng.integers(0, K))] = float(rng.choice([np.nan, np.inf, -np.inf]))
        assert np.array_equal(run(sess, layer, x, N, K)[kept], first[kept])
    assert np.array_equal(run(sess, layer, rows_of(a, kind), N, K), first)
    layer.close()


def test_passes_over_long_k_repeat_bit_for_bit(sess):
    """Eight rows of bf16 x 4096 x 14336: sixteen waves a workgroup, which load twice.  Layers in turn, nothing waiting in between."""
    rng = np.random.default_rng(14)
    M, N, K, group = 8, 4096, 14336, 128
    layers = [Layer(sess, rng, N, K, group, exact=False) for _ in range(2)]
    x = [rows_of(rng.standard_normal((M, K)) * np.where(rng.random((M, K)) < 0.005, 20, 1), "bf16") for _ in layers]
    ws = ops.G4Workspace(sess, M, K, N)
    outs = [torch.zeros((M, N), device="cuda") for _ in layers]
    first = None
    for turn in range(40):
        for c in outs:
            c.fill_(77)
        ready()
        for _ in range(3):
            for layer, a, c in zip(layers, x, outs):
                ws.run(layer.w, a, c)
        done(sess)
        if first is None:
            first = [c.clone() for c in outs]
            for layer, a, c in zip(layers, x, first):
                want = host(a) @ layer.values.T
                assert (np.abs(host(c) - want) <= ref.sum_bound(host(a), layer.sizes, K) + ref.HALF_STEP["f32"] * np.abs(want)).all()
        assert all(torch.equal(a, b) for a, b in zip(first, outs)), turn
    for h in (ws, *layers):
        h.close()
