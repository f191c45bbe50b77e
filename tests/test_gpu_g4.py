"""GPU tests of the group-scaled 4-bit layers through the C ABI, against their definition in 64 bits (g4_reference).

Products are compared bit for bit where fp32 holds every sum exactly in any order (small integers, scales that are powers of two); others may be off by
sum_bound, which counts the additions that a term goes through.
"""
import ctypes as C

import numpy as np
import pytest
import torch

from rknpu2_matmul_open_amd import capi, ops
from tests import g4_reference as ref
from tests.test_gpu_mx4 import TYPES, device, done, host, poisoned, ready, untouched

pytestmark = pytest.mark.gpu

HALVES = {"f16": torch.float16, "bf16": torch.bfloat16}


class Layer:
    """A seeded matrix.  exact: scales are +-1/2, 1, 2 and zero points up to 16."""

    def __init__(self, sess, rng, N, K, group, gate_up=False, exact=True, kind="f16", zeros=True):
        groups = -(-K // group)
        self.code = rng.integers(0, 16, (N, K))
        self.zeros = rng.integers(0, 17 if exact else 256, (N, groups)).astype(np.uint8) if zeros else None
        s = rng.choice([0.5, 1.0, -1.0, 2.0], (N, groups)) if exact else rng.standard_normal((N, groups)) * np.exp2(rng.integers(-12, -4, (N, groups)))
        if not exact and zeros:
            self.zeros[rng.random((N, groups)) < 0.9] %= 16
        t = device(s, kind)
        self.scales, self.group = host(t), group
        packed = ref.pack(self.code)
        if K % 2:
            packed[:, -1] |= 0xa0 # (what is beyond a row counts for nothing)
        codes = device(packed)
        ready()
        self.w = ops.G4Weights.from_device(sess, K, N, group, codes, t, None if self.zeros is None else device(self.zeros), gate_up=gate_up)
        self.values, self.sizes = (f(self.code, self.scales, self.zeros, group) for f in (ref.weights, ref.sizes))

    def close(self):
        self.w.close()


def rows_of(x, kind, pad=0, shift=0):
    """x on the device, rows `pad` values further apart than they are long, `shift` values behind an aligned address; NaN around them."""
    M, K = x.shape
    whole = torch.full((M * (K + pad) + shift + 8,), float("nan"), dtype=HALVES[kind], device="cuda")
    view = whole[shift:shift + M * (K + pad)].view(M, K + pad)[:, :K]
    view.copy_(device(x, kind))
    return view


@pytest.mark.parametrize("M,N,K,group", ref.SHAPES)
def test_product_of_small_integers_bit_for_bit(sess, M, N, K, group):
    rng = np.random.default_rng(M * 7 + N * 3 + K)
    layer = Layer(sess, rng, N, K, group, kind="bf16" if K % 2 else "f16", zeros=N % 3 != 0)
    a = rng.integers(-4, 5, (M, K)).astype(np.float64)
    want = a @ layer.values.T
    assert 2 * (np.abs(a) @ layer.sizes.T).max() < 2 ** 24 # (multiples of 1/2: exact in any order)
    ws = ops.G4Workspace(sess, M, K, N)
    for kind, out, pad_a, shift, pad_c in (("f16", "f32", 0, 0, 0), ("bf16", "f16", 3, 1, 5), ("f16", "bf16", 8, 3, 0), ("bf16", "f32", 0, 0, 1)):
        x = rows_of(a, kind, pad_a, shift)
        c, buf = poisoned(M, N, out, N + pad_c)
        ready()
        ws.run(layer.w, x, c)
        done(sess)
        with np.errstate(over="ignore"):
            rounded = torch.from_numpy(want.astype(np.float32)).to(TYPES[out]).double().numpy()
        got = host(c)
        assert np.array_equal(got, rounded), (kind, out, np.argwhere(got != rounded)[:5], np.abs(got - rounded).max())
        assert untouched(buf, M, N, N + pad_c)
    ws.close()
    layer.close()


def row_bound(x, layer_sizes, K):
    """sum_bound, and what staged rows of bf16 lose: half of 2^-38 of a row's largest value."""
    return ref.sum_bound(x, layer_sizes, K) + 2.0 ** -39 * np.abs(x).max(1)[:, None] * layer_sizes.sum(1)[None, :]


@pytest.mark.parametrize("M,N,K,group", [s for i, s in enumerate(ref.SHAPES) if i % 2 == 0])
def test_product_of_ordinary_rows_within_fp32_sums(sess, M, N, K, group):
    rng = np.random.default_rng(M + N + K)
    layer = Layer(sess, rng, N, K, group, exact=False, kind="f16" if M % 2 else "bf16")
    ws = ops.G4Workspace(sess, M, K, N)
    for kind, out, power in (("f16", "f32", 0), ("bf16", "f32", 100), ("bf16", "bf16", -60)):
        x = rows_of(rng.standard_normal((M, K)) * np.exp2(rng.integers(-12, 1, (M, 1)) + power), kind)
        c, buf = poisoned(M, N, out)
        ready()
        ws.run(layer.w, x, c)
        done(sess)
        a = host(x)
        want, bound = a @ layer.values.T, row_bound(a, layer.sizes, K)
        far = np.abs(host(c) - want) - bound - ref.HALF_STEP[out] * (np.abs(want) + bound)
        assert far.max() <= 0, (kind, out, far.max())
        assert untouched(buf, M, N, N)
    ws.close()
    layer.close()


@pytest.mark.parametrize("M", [1, 7, 16, 17, 100, 300])
def test_rows_of_every_size_and_bad_ones_are_independent(sess, M):
    """Rows from fp32's smallest numbers to bf16's largest, zeros, and rows that hold an infinity or a NaN beside them."""
    rng = np.random.default_rng(M)
    N, K = 70, 264
    layer = Layer(sess, rng, N, K, 32)
    a = rng.integers(-4, 5, (M, K)) * np.exp2(rng.choice([-130, -126, -100, 0, 60, 112], (M, 1)))
    a[::5] = 0.0
    bad = np.zeros(M, bool)
    x = rows_of(a, "bf16")
    if M > 1:
        for r, v in ((1, np.nan), (M // 2, np.inf), (M - 1, -np.inf)):
            x[r, int(rng.integers(0, K))] = float(v)
            bad[r] = True
    ws = ops.G4Workspace(sess, M, K, N)
    c, buf = poisoned(M, N, "f32")
    ready()
    ws.run(layer.w, x, c)
    done(sess)
    want = (a @ layer.values.T).astype(np.float32)
    got = host(c)
    assert np.array_equal(got[~bad], want[~bad].astype(np.float64)), np.argwhere(got[~bad] != want[~bad])[:5]
    assert not np.isfinite(got[bad]).any()
    assert untouched(buf, M, N, N)
    ws.close()
    layer.close()


@pytest.mark.parametrize("M", [3, 16, 40, 200])
def test_fp16_rows_of_subnormals_and_of_the_largest(sess, M):
    """fp16 rows are multiplied as they are: subnormals and 65504 beside each other, one value of K each, exact."""
    rng = np.random.default_rng(M)
    N, K = 96, 256
    layer = Layer(sess, rng, N, K, 64)
    a = np.zeros((M, K))
    a[np.arange(M), rng.integers(0, K, M)] = np.resize([2.0 ** -24, 65504, -3 * 2.0 ** -24, 1023 * 2.0 ** -24, -65504], M)
    ws = ops.G4Workspace(sess, M, K, N)
    x, c = rows_of(a, "f16"), torch.zeros((M, N), device="cuda")
    ready()
    ws.run(layer.w, x, c)
    done(sess)
    assert np.array_equal(host(c), a @ layer.values.T)
    ws.close()
    layer.close()


@pytest.mark.parametrize("M", [1, 20, 300])
def test_every_code_and_zero_point_reads_back(sess, M):
    """One-hot rows give the matrix itself, rounded once from fp32 where a scale of fp16 or bf16 times an integer up to 255 is exact."""
    K, N, group = 512, 256, 32
    code = (np.arange(K)[None, :] + np.arange(N)[:, None]) % 16
    zeros = ((np.arange(K // group)[None, :] * N + np.arange(N)[:, None]) % 256).astype(np.uint8)
    for kind in HALVES:
        s = device(np.random.default_rng(1).standard_normal((N, K // group)) * 0.01, kind)
        at = device(zeros)
        ready()
        w = ops.G4Weights.from_device(sess, K, N, group, device(ref.pack(code)), s, at)
        ws = ops.G4Workspace(sess, 300, K, N)
        for start in range(0, 600, 300):
            x = torch.zeros((M, K), dtype=torch.float16, device="cuda")
            which = (np.arange(M) + start) % K
            x[torch.arange(M), torch.from_numpy(which)] = 1.0
            c = torch.zeros((M, N), device="cuda")
            ready()
            ws.run(w, x, c)
            done(sess)
            assert np.array_equal(host(c), ref.weights(code, host(s), zeros, group)[:, which].T)
        ws.close()
        w.close()


@pytest.mark.parametrize("gate_up", [False, True])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_weights_from_host_arrays_are_those_from_the_device(sess, gate_up, kind):
    rng = np.random.default_rng(5)
    N, K, group, M = 70, 99, 64, 20
    layer = Layer(sess, rng, N, K, group, gate_up=gate_up, kind=kind)
    scales = layer.scales.astype(np.float16) if kind == "f16" else (layer.scales.astype(np.float32).view(np.uint32) >> 16).astype(np.uint16)
    w = ops.G4Weights(sess, K, N, group, ref.pack(layer.code), scales, layer.zeros, gate_up=gate_up, scale_type=None if kind == "f16" else capi.MX4_BF16)
    config, size = capi.G4WeightConfig(), C.c_uint64(0)
    assert sess.lib.rk_npu_g4_weights_query(w.h, C.byref(config), C.byref(size)) == 0
    assert (config.K, config.N, config.group, config.gate_up, config.scale_type) == (K, N, group, int(gate_up), capi.MX4_F16 if kind == "f16" else capi.MX4_BF16)
    assert N * K / 2 <= size.value <= 4 * 128 * 128
    x = rows_of(rng.standard_normal((M, K)), "bf16")
    ws, run = ops.G4Workspace(sess, M, K, N), []
    for which in (layer.w, w):
        c = torch.zeros((M, N // 2 if gate_up else N), device="cuda")
        ready()
        (ws.run_swiglu if gate_up else ws.run)(which, x, c)
        done(sess)
        run.append(c)
    assert torch.equal(*run)
    for h in (ws, w, layer):
        h.close()


@pytest.mark.parametrize("M,N,K", [(8, 200, 4096), (40, 700, 4096), (300, 300, 14336)])
def test_results_do_not_depend_on_the_workspace_or_on_other_rows(sess, M, N, K):
    rng = np.random.default_rng(M)
    layer = Layer(sess, rng, N, K, 128, exact=False)
    x = rows_of(rng.standard_normal((M, K)), "f16")
    out = []
    for rows, most in ((M, N), (M + 1000, N + 5000), (M, N)):
        ws, c = ops.G4Workspace(sess, rows, K, most), torch.zeros((M, N), device="cuda")
        ready()
        ws.run(layer.w, x, c)
        done(sess)
        ws.close()
        out.append(c)
    assert torch.equal(out[0], out[1]) and torch.equal(out[0], out[2])
    layer.close()


# ---- SwiGLU ------------------------------------------------------------------------------


@pytest.mark.parametrize("M,F,K,group", ref.SWIGLU)
def test_swiglu(sess, M, F, K, group):
    """Off by the sums' bounds through silu, whose slope is below 1.1, and the exponential, the reciprocal and the products: together below 2^-19 of the result."""
    rng = np.random.default_rng(M + F + K)
    layer = Layer(sess, rng, 2 * F, K, group, gate_up=True, exact=False, kind="bf16" if F % 2 else "f16")
    ws = ops.G4Workspace(sess, M, K, 2 * F)
    for kind, out, pad in (("f16", "f32", 0), ("bf16", "bf16", 3), ("bf16", "f16", 0)):
        x = rows_of(rng.standard_normal((M, K)), kind)
        c, buf = poisoned(M, F, out, F + pad)
        ready()
        ws.run_swiglu(layer.w, x, c)
        done(sess)
        a = host(x)
        s, e = a @ layer.values.T, row_bound(a, layer.sizes, K)
        gate, up, eg, eu = s[:, :F], s[:, F:], e[:, :F], e[:, F:]
        silu = ref.silu(gate)
        want, bound = silu * up, 1.1 * eg * (np.abs(up) + eu) + np.abs(silu) * eu + 2.0 ** -19 * np.abs(silu * up) + 1e-30
        with np.errstate(invalid="ignore"):
            far = np.abs(host(c) - want) - bound - ref.HALF_STEP[out] * (np.abs(want) + bound) - ref.LEAST[out]
        far[(out == "f16") & (np.abs(want) > 65000)] = 0
        assert far.max() <= 0, (kind, out, far.max())
        assert untouched(buf, M, F, F + pad)
    ws.close()
    layer.close()


@pytest.mark.parametrize("M", [1, 16, 20, 100])
def test_swiglu_of_far_gates(sess, M):
    """One-hot rows: exact sums over the whole range of the exponential; 16 roundings or ulps around it."""
    K = F = 512
    gates = np.array([0, 1, -1, 2, -2, 8, -8, 16, -24, 48, -64, 88, -88, 120, -128, -192])
    code, scales, zeros = np.full((2 * F, K), 8), np.ones((2 * F, K // 32)), np.full((2 * F, K // 32), 8, np.uint8)
    at = np.arange(F)
    code[at, at] = np.where(np.abs(gates)[at % 16] > 7, 8 + np.sign(gates[at % 16]), 8 + gates[at % 16])
    scales[at, at // 32] = np.where(np.abs(gates[at % 16]) > 7, np.abs(gates[at % 16]), 1)
    code[F + at, at] = 8 + at % 3 + 1
    w = ops.G4Weights(sess, K, 2 * F, 32, ref.pack(code), scales.astype(np.float16), zeros, gate_up=True)
    values = ref.weights(code, scales, zeros, 32)
    a = np.zeros((M, K))
    a[np.arange(M), np.random.default_rng(M).integers(0, K, M)] = 1.0
    ws, x, c = ops.G4Workspace(sess, M, K, 2 * F), rows_of(a, "bf16"), torch.zeros((M, F), device="cuda")
    ready()
    ws.run_swiglu(w, x, c)
    done(sess)
    want = ref.silu(a @ values[:F].T) * (a @ values[F:].T)
    assert (np.abs(host(c) - want) <= 16 * 2.0 ** -24 * np.abs(want) + 1e-36).all()
    ws.close()
    w.close()


# ---- calls ---------------------------------------------------------------------------------


@pytest.mark.parametrize("M,kind", [(5, "bf16"), (5, "f16"), (30, "f16"), (30, "bf16"), (200, "bf16")])
def test_product_between_the_slices_of_a_buffer(sess, M, kind):
    """Input and output are columns of one buffer, in either order."""
    rng = np.random.default_rng(M)
    N, K = 70, 128
    layer = Layer(sess, rng, N, K, 32)
    a = rng.integers(-4, 5, (M, K)).astype(np.float64)
    ws = ops.G4Workspace(sess, M, K, N)
    for x_at, c_at in ((0, 130), (72, 1)):
        whole = torch.full((M, 208), 77.0, dtype=HALVES[kind], device="cuda")
        whole[:, x_at:x_at + K].copy_(device(a, kind))
        ready()
        ws.run(layer.w, whole[:, x_at:x_at + K], whole[:, c_at:c_at + N])
        done(sess)
        want = np.full((M, 208), 77.0)
        want[:, x_at:x_at + K] = a
        want[:, c_at:c_at + N] = host(torch.from_numpy(a @ layer.values.T).to(HALVES[kind]))
        assert np.array_equal(host(whole), want)
    ws.close()
    layer.close()


@pytest.mark.parametrize("M,N,K,gate_up", [(1, 100, 4096, False), (3, 40, 1001, True), (50, 700, 4096, False), (64, 500, 4096, True), (200, 300, 500, True)])
def test_captured_calls_replay_what_the_eager_call_gives(sess, M, N, K, gate_up):
    """Two graphs of one workspace, replayed in turn with new rows and with eager work of other rows in between."""
    rng = np.random.default_rng(M + K)
    layers = [Layer(sess, rng, 2 * N if gate_up else N, K, 64, gate_up=gate_up, exact=False) for _ in range(2)]
    ws = ops.G4Workspace(sess, M, K, 2 * N if gate_up else N)
    run = ws.run_swiglu if gate_up else ws.run
    x, other = rows_of(rng.standard_normal((M, K)), "bf16"), rows_of(rng.standard_normal((M, K)), "bf16")
    outs, scrap = [torch.zeros((M, N), device="cuda") for _ in range(2)], torch.zeros((M, N), device="cuda")
    ready()
    graphs = []
    for layer, c in zip(layers, outs):
        run(layer.w, x, c)
        done(sess)
        assert sess.lib.rk_npu_hip_capture_begin(sess.ctx) == 0
        run(layer.w, x, c)
        graphs.append(sess.lib.rk_npu_hip_capture_end(sess.ctx))
        assert graphs[-1]
    for turn in range(4):
        x.copy_(device(rng.standard_normal((M, K)), "bf16"))
        want = []
        ready()
        for layer in layers:
            c = torch.zeros((M, N), device="cuda")
            ready()
            run(layer.w, x, c)
            done(sess)
            want.append(c)
        for c in outs:
            c.fill_(-1)
        ready()
        for i in ((0, 1), (1, 0))[turn % 2]:
            assert sess.lib.rk_npu_hip_graph_launch(sess.ctx, graphs[i]) == 0
            run(layers[i].w, other, scrap)
        done(sess)
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    for graph in graphs:
        sess.lib.rk_npu_hip_graph_free(graph)
    for h in (ws, *layers):
        h.close()


def test_zero_rows_write_nothing(sess):
    rng = np.random.default_rng(1)
    layer = Layer(sess, rng, 64, 96, 32)
    ws, c = ops.G4Workspace(sess, 8, 96, 64), torch.full((8, 64), 5.0, device="cuda")
    ready()
    ws.run(layer.w, torch.zeros((0, 96), dtype=torch.float16, device="cuda"), c[:0])
    done(sess)
    assert (host(c) == 5).all()
    ws.close()
    layer.close()


def test_refusals(sess):
    rng = np.random.default_rng(2)
    K, N = 96, 64
    layer, pair = Layer(sess, rng, N, K, 32), Layer(sess, rng, N, K, 32, gate_up=True)
    ws, small, short = ops.G4Workspace(sess, 8, K, N), ops.G4Workspace(sess, 8, K, N - 1), ops.G4Workspace(sess, 8, K - 1, N)
    x, c = torch.ones((8, 128), dtype=torch.float16, device="cuda"), torch.full((8, 128), 5.0, device="cuda")
    ready()
    lib, bad = sess.lib, capi.RK_NPU_ERR_PARAM
    p, q = x.data_ptr(), c.data_ptr()
    run = lambda ws=ws, w=layer.w, rows=4, at=1, a=p, lda=128, ct=0, out=q, ldc=128: lib.rk_npu_g4_run_device(ws.h, w.h, rows, at, a, lda, ct, out, ldc)  # noqa: E731
    assert run() == 0
    done(sess)
    for wrong in (dict(rows=-1), dict(rows=9), dict(at=0), dict(at=3), dict(at=-1), dict(ct=3), dict(ct=-1), dict(a=None), dict(out=None), dict(lda=K - 1), dict(ldc=N - 1),
                  dict(a=p + 1), dict(out=q + 2), dict(ct=1, out=q + 1), dict(w=pair.w), dict(ws=small), dict(ws=short), dict(out=p), dict(ct=1, out=p + 2 * 3 * 128),
                  dict(ct=1, out=p + 2 * 95), dict(lda=1 << 62), dict(ldc=1 << 62)):
        assert run(**wrong) == bad, wrong
    assert run(ct=1, out=p + 2 * 96, ldc=128, rows=1) == 0 # (beside the row)
    done(sess)
    assert lib.rk_npu_g4_run_swiglu_device(ws.h, layer.w.h, 4, 1, p, 128, 0, q, 128) == bad
    assert lib.rk_npu_g4_run_device(None, layer.w.h, 4, 1, p, 128, 0, q, 128) == bad and lib.rk_npu_g4_run_device(ws.h, None, 4, 1, p, 128, 0, q, 128) == bad
    codes, scales = ref.pack(layer.code), layer.scales.astype(np.float16)
    create = lambda K=96, N=64, group=32, gate_up=0, kind=1, p=codes.ctypes.data, s=scales.ctypes.data: lib.rk_npu_g4_weights_create(  # noqa: E731
        sess.domain, C.byref(capi.G4WeightConfig(K, N, group, gate_up, kind)), p, s, None)
    for wrong in (dict(K=0), dict(K=-1), dict(K=1 << 30), dict(N=0), dict(N=-1), dict(N=2 ** 31 - 1), dict(N=63, gate_up=1), dict(group=0), dict(group=-32), dict(group=16),
                  dict(group=48), dict(kind=0), dict(kind=3), dict(p=None), dict(s=None), dict(s=scales.ctypes.data + 1)):
        assert not create(**wrong), wrong
    for rows, k, n in ((0, 96, 64), (-1, 96, 64), (8, 0, 64), (8, 96, 0), (8, 1 << 30, 64), (2 ** 31 - 1, 96, 64), (8, 96, 2 ** 31 - 1)):
        assert not lib.rk_npu_g4_workspace_create(sess.domain, rows, k, n)
    other = lib.rk_npu_iommu_domain_create(sess.ctx, 3)
    foreign = lib.rk_npu_g4_workspace_create(other, 8, K, N)
    assert foreign and lib.rk_npu_g4_run_device(foreign, layer.w.h, 4, 1, p, 128, 0, q, 128) == capi.RK_NPU_ERR_DOMAIN
    lib.rk_npu_g4_workspace_free(foreign)
    lib.rk_npu_iommu_domain_free(other)
    for h in (ws, small, short, layer, pair):
        h.close()


def test_out_of_memory_at_every_allocation(sess):
    code = np.zeros((64, 48), np.uint8)
    scales, zeros, lib = np.ones((64, 3), np.float16), np.zeros((64, 3), np.uint8), sess.lib
    config = capi.G4WeightConfig(96, 64, 32, 0, 1)
    create = lambda: lib.rk_npu_g4_weights_create(sess.domain, C.byref(config), code.ctypes.data, scales.ctypes.data, zeros.ctypes.data)  # noqa: E731
    for n in (1, 2, 3, 4, 5):
        lib.rk_npu_hip_fail_alloc_after(n)
        assert not create(), n
    for n in (1, 2, 3):
        lib.rk_npu_hip_fail_alloc_after(n)
        assert not lib.rk_npu_g4_workspace_create(sess.domain, 128, 8192, 64), n
    lib.rk_npu_hip_fail_alloc_after(0)
    w = create()
    assert w
    lib.rk_npu_g4_weights_free(w)


@pytest.mark.parametrize("M,kind", [(4, "bf16"), (40, "f16"), (40, "bf16")])
def test_rows_further_apart_than_32_bits(sess, M, kind):
    """The last row begins more than 2^32 bytes behind the first; fp16 rows of tiles this far apart are staged."""
    K, N = 128, 64
    ld = (1 << 31) // M + 128 + (-(1 << 31) // M) % 128
    if torch.cuda.mem_get_info()[0] < ld * M * 2 + (1 << 33):
        pytest.skip("no room")
    rng = np.random.default_rng(M)
    layer = Layer(sess, rng, N, K, 64)
    a = rng.integers(-4, 5, (M, K)).astype(np.float64)
    whole = torch.empty(((M - 1) * ld + K) + 8, dtype=HALVES[kind], device="cuda")
    x = whole.as_strided((M, K), (ld, 1))
    x.copy_(device(a, kind))
    out = torch.empty((M - 1) * ld + N, dtype=HALVES[kind], device="cuda").as_strided((M, N), (ld, 1))
    ws = ops.G4Workspace(sess, M, K, N)
    ready()
    ws.run(layer.w, x, out)
    done(sess)
    assert np.array_equal(host(out), host(torch.from_numpy(a @ layer.values.T).to(HALVES[kind])))
    ws.close()
    layer.close()


def test_two_threads(sess):
    """With a workspace each, both get their products; with one, a call is made or refused as BUSY, and nothing else."""
    import threading
    rng = np.random.default_rng(8)
    M, N, K = 40, 200, 1000
    layer = Layer(sess, rng, N, K, 64)
    a = [rng.integers(-4, 5, (M, K)).astype(np.float64) for _ in range(2)]
    x = [rows_of(v, "bf16") for v in a]
    for shared in (False, True):
        spaces = [ops.G4Workspace(sess, M, K, N) for _ in range(2)]
        outs, codes = [torch.zeros((M, N), device="cuda") for _ in range(2)], [set(), set()]
        ready()

        def loop(i):
            ws = spaces[0 if shared else i]
            for _ in range(200):
                codes[i].add(sess.lib.rk_npu_g4_run_device(ws.h, layer.w.h, M, capi.MX4_BF16, x[i].data_ptr(), x[i].stride(0), capi.MX4_F32, outs[i].data_ptr(), N))
        threads = [threading.Thread(target=loop, args=(i,)) for i in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        done(sess)
        for i in range(2):
            assert codes[i] <= ({0, capi.RK_NPU_ERR_BUSY} if shared else {0})
            if 0 in codes[i]:
                assert np.array_equal(host(outs[i]), a[i] @ layer.values.T)
        for ws in spaces:
            ws.close()
    layer.close()
