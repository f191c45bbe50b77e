"""GPU tests of the ways through the MX4 kernels that only some sizes take: workgroups that multiply several 256 x 256 tiles with more than one
group of 512 k each, gate / up products with K in parts, and rows that the few-row kernel norms itself.

Which way a size takes is arithmetic (rkh_mx4_route, rkh_mx4_takes_rows) and asserted first.  Products of exact_rows are compared bit for bit
with products in 64 bits, others within the bounds of test_gpu_mx4; a call that stands for several with the several, bit for bit.
"""
import numpy as np
import pytest
import torch

from rknpu2_matmul_open_amd import ops
from tests import mx4_reference as ref
from tests.test_gpu_mx4 import HALF_STEP, TYPES, Layer, device, done, host, ordinary, poisoned, ready, route, untouched

pytestmark = pytest.mark.gpu

CUS = 256


def tiles(sess, M, N, K, swiglu=0):
    """(whole 256 x 256 tiles, what goes as halves) of a product that takes them."""
    kernel, rows, columns, parts = route(sess, M, N, K, swiglu)
    assert (kernel, rows, columns, parts) == (1, 256, 256, 1)
    places = 2 * (-(-N // 32) * 32) if swiglu else -(-N // 32) * 32
    count = -(-M // 256) * -(-places // 256)
    left = count % CUS
    return (count - left, left) if left <= CUS // 2 else (count, 0)


def product64(a, values):
    """A product in 64 bits, on the device."""
    return a @ values.t().contiguous()


def device64(x):
    return torch.from_numpy(np.ascontiguousarray(x)).to("cuda")


# ---- tile after tile -----------------------------------------------------------------------

# (M, N, K; whole tiles of the busiest workgroup, whether halves follow)
CHAINS = [(4200, 8300, 1100, 2, True), (5000, 6200, 2050, 2, False), (6000, 9000, 600, 3, True)]


@pytest.mark.parametrize("M,N,K,chain,halves", CHAINS)
def test_chained_tiles_of_several_groups_bit_for_bit(sess, M, N, K, chain, halves):
    whole, rest = tiles(sess, M, N, K)
    assert -(-whole // CUS) == chain and (rest > 0) == halves and -(-K // 512) >= 2 and K % 512
    rng = np.random.default_rng(M)
    layer = Layer(sess, rng, N, K)
    a = ref.values(*ref.exact_rows(rng, M, K), K)
    want = product64(device64(a), device64(layer.values))
    ws = ops.MX4Workspace(sess, M, K, N)
    x = device(a, "bf16")
    for out, pad in (("f32", 0), ("f16", 5), ("bf16", 0)):
        c, buf = poisoned(M, N, out, N + pad)
        ready()
        ws.run(layer.w, x, c)
        done(sess)
        assert torch.equal(c, want.to(TYPES[out])), out
        assert untouched(buf, M, N, N + pad)
    ws.close()
    layer.close()


@pytest.mark.parametrize("M,F,K,halves", [(1200, 11008, 1100, False), (3060, 6490, 600, True)])
def test_chained_tiles_with_swiglu(sess, M, F, K, halves):
    whole, rest = tiles(sess, M, F, K, 1)
    assert whole > CUS and (rest > 0) == halves
    rng = np.random.default_rng(M)
    layer = Layer(sess, rng, 2 * F, K, gate_up=True, make=ordinary)
    d = device(rng.standard_normal((M, K)), "f32")
    a, g, u = device64(ref.round_trip(host(d))), device64(layer.values[:F]), device64(layer.values[F:])
    gate, up = product64(a, g), product64(a, u)
    silu = gate / (1 + torch.exp(-gate))
    want = silu * up
    eg, eu = (K * 2.0 ** -24 * product64(a.abs(), v.abs()) for v in (g, u))
    bound = 1.1 * eg * (up.abs() + eu) + silu.abs() * eu + 2.0 ** -19 * want.abs() + 1e-30 # (swiglu_bound of test_gpu_mx4)
    ws = ops.MX4Workspace(sess, M, K, 2 * F)
    for out, pad in (("f32", 0), ("bf16", 3)):
        c, buf = poisoned(M, F, out, F + pad)
        ready()
        ws.run_swiglu(layer.w, d, c)
        done(sess)
        assert ((c.double() - want).abs() <= bound + HALF_STEP[out] * (want.abs() + bound)).all(), out
        assert untouched(buf, M, F, F + pad)
    ws.close()
    layer.close()


def ffn_is_its_two_calls(sess, M, H, F):
    rng = np.random.default_rng(M + H + F)
    gu, dn = Layer(sess, rng, 2 * F, H, gate_up=True, make=ordinary), Layer(sess, rng, H, F, make=ordinary)
    gws, dws = ops.MX4Workspace(sess, M, H, 2 * F), ops.MX4Workspace(sess, M, F, H)
    x = device(rng.standard_normal((M, H)), "f32")
    middle, two, one = (torch.zeros((M, n), device="cuda") for n in (F, H, H))
    full = torch.ones((M, F), device="cuda")
    ready()
    dws.run(dn.w, full, two) # (what the down workspace holds beforehand would show)
    ops.mx4_ffn(gws, gu.w, dws, dn.w, x, one)
    gws.run_swiglu(gu.w, x, middle)
    dws.run(dn.w, middle, two)
    done(sess)
    assert torch.equal(one, two) and torch.isfinite(one).all() and one.abs().max() > 0
    a = ref.round_trip(host(middle))
    got, want, size = host(two), product64(device64(a), device64(dn.values)).cpu().numpy(), product64(device64(np.abs(a)), device64(np.abs(dn.values))).cpu().numpy()
    assert (np.abs(got - want) <= F * 2.0 ** -24 * size + 2.0 ** -24 * np.abs(want)).all()
    for h in (gws, dws, gu, dn):
        h.close()


@pytest.mark.parametrize("M,H,F", [(1200, 1100, 11008), (3060, 600, 6490)])
def test_ffn_of_chained_tiles_is_its_two_calls_bit_for_bit(sess, M, H, F):
    assert tiles(sess, M, F, H, 1)[0] > CUS
    ffn_is_its_two_calls(sess, M, H, F)


def test_captured_chains_replay_what_the_eager_call_gives(sess):
    """The rows change between replays, and the eager call goes through the same workspace in between."""
    M, N, K = 4200, 8300, 600
    assert tiles(sess, M, N, K)[0] > CUS
    rng = np.random.default_rng(3)
    layer = Layer(sess, rng, N, K, make=ordinary)
    ws = ops.MX4Workspace(sess, M, K, N)
    inputs = [device(rng.standard_normal((M, K)), "bf16") for _ in range(3)]
    x, got, eager = inputs[0].clone(), torch.zeros((M, N), dtype=torch.float16, device="cuda"), torch.zeros((M, N), dtype=torch.float16, device="cuda")
    ready()
    ws.run(layer.w, x, got)
    done(sess)
    assert sess.lib.rk_npu_hip_capture_begin(sess.ctx) == 0
    ws.run(layer.w, x, got)
    graph = sess.lib.rk_npu_hip_capture_end(sess.ctx)
    assert graph
    for source in inputs + inputs[:2]:
        x.copy_(source)
        got.zero_()
        ready()
        assert sess.lib.rk_npu_hip_graph_launch(sess.ctx, graph) == 0
        ws.run(layer.w, source, eager)
        done(sess)
        assert torch.equal(got, eager) and got.abs().max() > 0
    sess.lib.rk_npu_hip_graph_free(graph)
    ws.close()
    layer.close()


# ---- gate / up products with K in parts ----------------------------------------------------


@pytest.mark.parametrize("M,F,K", [(40, 256, 8192), (100, 350, 14336), (33, 33, 8200), (300, 128, 16384)])
def test_swiglu_with_k_in_parts(sess, M, F, K):
    assert route(sess, M, F, K, 1)[0] == 1 and route(sess, M, F, K, 1)[3] > 1
    rng = np.random.default_rng(M + F)
    layer = Layer(sess, rng, 2 * F, K, gate_up=True, make=ordinary)
    d = device(rng.standard_normal((M, K)), "f32")
    a, g, u = device64(ref.round_trip(host(d))), device64(layer.values[:F]), device64(layer.values[F:])
    gate, up = product64(a, g), product64(a, u)
    silu = gate / (1 + torch.exp(-gate))
    want = silu * up
    eg, eu = (K * 2.0 ** -24 * product64(a.abs(), v.abs()) for v in (g, u))
    bound = 1.1 * eg * (up.abs() + eu) + silu.abs() * eu + 2.0 ** -19 * want.abs() + 1e-30
    ws = ops.MX4Workspace(sess, M, K, 2 * F)
    for out, pad in (("f32", 0), ("bf16", 3), ("f16", 1)):
        c, buf = poisoned(M, F, out, F + pad)
        ready()
        ws.run_swiglu(layer.w, d, c)
        done(sess)
        assert ((c.double() - want).abs() <= bound + HALF_STEP[out] * (want.abs() + bound) + (2.0 ** -25 if out == "f16" else 0)).all(), out
        assert untouched(buf, M, F, F + pad)
    ws.close()
    layer.close()


@pytest.mark.parametrize("M,H,F", [(70, 8200, 300), (40, 14336, 130), (200, 8192, 64)])
def test_ffn_with_k_in_parts_is_its_two_calls_bit_for_bit(sess, M, H, F):
    assert route(sess, M, F, H, 1)[3] > 1
    ffn_is_its_two_calls(sess, M, H, F)


# ---- rows that the few-row kernel norms itself -----------------------------------------------

# one and several segments of 512, waves and groups of a wave; pieces fetched ahead and behind; K not a multiple of 512
FUSED = [(1, 64), (4, 72), (1, 4096), (3, 4096), (4, 2056), (2, 8192), (1, 4104), (1, 12296), (1, 16384), (3, 1000)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,H", FUSED)
def test_block_that_norms_its_rows_itself_is_its_calls_bit_for_bit(sess, M, H, kind):
    """The norm, the gate / up product on its rows, the down product and the norm behind it as calls of their own."""
    F = 200
    assert sess.lib.rkh_mx4_takes_rows(M, F, H, 1)
    rng = np.random.default_rng(M + H)
    gu, dn = Layer(sess, rng, 2 * F, H, gate_up=True, make=ordinary), Layer(sess, rng, H, F, make=ordinary)
    gws, dws = ops.MX4Workspace(sess, M, H, 2 * F), ops.MX4Workspace(sess, M, F, H)
    stream = torch.full((M, H + 3), 9.0, dtype=TYPES[kind], device="cuda")[:, :H] # (rows whose start is aligned to the type alone)
    stream.copy_(device(rng.standard_normal((M, H)) * np.exp2(rng.integers(-4, 4, (M, 1))), kind))
    branch, middle = torch.zeros((M, H), device="cuda"), torch.zeros((M, F), device="cuda")
    outs = [torch.zeros((M, H), dtype=TYPES[kind], device="cuda") for _ in range(2)]
    for weight in (None, device(1 + 0.2 * rng.standard_normal(H), "f32")):
        ready()
        ops.mx4_ffn_block(gws, gu.w, dws, dn.w, stream, branch, weight=weight, eps=1e-4, stream_out=outs[0])
        done(sess)
        whole = branch.clone()
        branch.zero_()
        ready()
        ops.block_norm(sess, stream, weight=weight, eps=1e-4, staged=gws)
        gws.run_staged(gu.w, middle)
        dws.run(dn.w, middle, branch)
        ops.block_norm(sess, stream, branch, stream_out=outs[1])
        done(sess)
        assert torch.equal(branch, whole) and torch.equal(*outs), weight is None
        assert torch.isfinite(whole).all() and (whole.abs().amax(dim=1) > 0).all()
    for h in (gws, dws, gu, dn):
        h.close()
