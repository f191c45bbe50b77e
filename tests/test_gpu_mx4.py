"""GPU tests of the MX4 rows and products through the C ABI, against the format's definition in 64 bits (mx4_reference).

Quantization is exact arithmetic and compared bit for bit.  Products are compared bit for bit on rows whose sums fp32 holds
exactly in any order (exact_rows); on others fp32 sums of n terms are off by at most n 2^-24 of the sum of magnitudes.
"""
import ctypes as C

import numpy as np
import pytest
import torch

from rknpu2_matmul_open_amd import capi, ops
from tests import mx4_reference as ref

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def device(x, kind=None):
    t = torch.from_numpy(np.ascontiguousarray(x))
    return (t if kind is None else t.to(TYPES[kind])).to("cuda")


def host(t):
    return t.detach().cpu().double().numpy()


def done(sess):
    assert sess.sync() == 0


def ready():
    torch.cuda.synchronize()  # (what torch has made on its own stream)


def poisoned(rows, columns, kind, pitch=None, extra=2):
    """A [rows, columns] view of rows `pitch` values apart, in a buffer of ones' bits; and the buffer."""
    pitch = pitch or columns
    buf = torch.full(((rows + extra) * pitch + 8,), 77.0, dtype=TYPES[kind], device="cuda")
    return buf[:rows * pitch].view(rows, pitch)[:, :columns], buf


def untouched(buf, rows, columns, pitch):
    """Everything but the rows is still 77."""
    whole = host(buf).copy()
    whole[:rows * pitch].reshape(rows, pitch)[:, :columns] = 77.0
    return (whole == 77.0).all()


def awkward(rng, rows, K):
    """Values of every size, with blocks of zeros, ties, subnormals and values that saturate."""
    x = rng.standard_normal((rows, K)) * np.exp2(rng.integers(-20, 14, (rows, 1)))
    flat = x.reshape(-1)
    flat[::97] = 0.0
    flat[5::131] = -0.0
    for r in range(rows):
        which = r % 6
        if which == 1:
            x[r] = rng.integers(-32, 33, K) / 4.0            # ties in every block
        elif which == 2:
            x[r] = 0.0
        elif which == 3:
            x[r] *= 2.0 ** -30 / max(1e-30, np.abs(x[r]).max()) # (subnormal in fp16)
    return x


# ---- rows --------------------------------------------------------------------------------


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,K,pad,shift", [(1, 1, 0, 0), (1, 32, 0, 0), (3, 31, 0, 0), (2, 33, 5, 1), (7, 64, 0, 0), (5, 4096, 0, 0), (6, 257, 3, 3), (67, 96, 1, 0),
                                              (300, 40, 0, 0)])
def test_quantize_and_back_bit_for_bit(sess, kind, rows, K, pad, shift):
    rng = np.random.default_rng(rows * 1000 + K)
    whole = torch.zeros(rows * (K + pad) + shift, dtype=TYPES[kind], device="cuda")
    x = whole[shift:].view(rows, K + pad)[:, :K]
    x.copy_(device(awkward(rng, rows, K), kind))
    blocks = -(-K // 32)
    codes, scales = (torch.full((rows + 1, w), 0xA5, dtype=torch.uint8, device="cuda") for w in (blocks * 16, blocks))
    back, buf = poisoned(rows, K, "f32", K + pad)
    ready()
    ops.mx4_quantize(sess, x, codes[:rows], scales[:rows])
    ops.mx4_dequantize(sess, codes[:rows], scales[:rows], back)
    done(sess)
    want_codes, want_scales = ref.quantize(host(x))
    assert np.array_equal(scales[:rows].cpu().numpy(), want_scales)
    assert np.array_equal(codes[:rows].cpu().numpy(), want_codes)
    assert (codes[rows:].cpu().numpy() == 0xA5).all() and (scales[rows:].cpu().numpy() == 0xA5).all()
    assert np.array_equal(host(back), ref.values(want_codes, want_scales, K).astype(np.float32))
    assert untouched(buf, rows, K, K + pad)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_blocks_with_infinities_and_nan(sess, kind):
    x = np.ones((4, 96))
    x[0, 3] = np.inf
    x[1, 40] = np.nan
    x[2, 95] = -np.inf
    d = device(x, kind)
    codes, scales = torch.zeros((4, 48), dtype=torch.uint8, device="cuda"), torch.zeros((4, 3), dtype=torch.uint8, device="cuda")
    y = torch.zeros((4, 96), device="cuda")
    ready()
    ops.mx4_quantize(sess, d, codes, scales)
    ops.mx4_dequantize(sess, codes, scales, y)
    done(sess)
    bad = np.zeros((4, 3), bool)
    bad[0, 0] = bad[1, 1] = bad[2, 2] = True
    assert np.array_equal(scales.cpu().numpy() == 255, bad)
    assert np.array_equal(np.isnan(host(y)), bad.repeat(32, 1)) and (host(y)[~bad.repeat(32, 1)] == 1).all()


def test_largest_and_smallest_fp32(sess):
    """Scales at both ends: the largest fp32 has 2^125, values below 2^-125 share 2^-127."""
    tops = [np.finfo(np.float32).max, 2.0 ** 127, 2.0 ** -126, 2.0 ** -149, 3 * 2.0 ** -128, 2.0 ** -124, 2.0 ** -125]
    x = np.zeros((len(tops), 32), np.float32)
    x[:, 0] = tops
    x[:, 1] = -np.array(tops) / 2
    d = device(x)
    codes, scales = (torch.zeros((len(tops), w), dtype=torch.uint8, device="cuda") for w in (16, 1))
    ready()
    ops.mx4_quantize(sess, d, codes, scales)
    done(sess)
    want = ref.quantize(x)
    assert np.array_equal(codes.cpu().numpy(), want[0]) and np.array_equal(scales.cpu().numpy(), want[1])


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_every_code_under_every_scale_reads_back(sess, kind):
    codes = np.tile(np.arange(16, dtype=np.uint8)[None, :] | (np.arange(15, -1, -1, dtype=np.uint8)[None, :] << 4), (256, 1))
    scales = np.arange(256, dtype=np.uint8)[:, None]
    y = torch.zeros((256, 32), dtype=TYPES[kind], device="cuda")
    dc, ds = device(codes), device(scales)
    ready()
    ops.mx4_dequantize(sess, dc, ds, y)
    done(sess)
    with np.errstate(over="ignore"):
        want = torch.from_numpy(ref.values(codes, scales, 32).astype(np.float32)).to(TYPES[kind]).double().numpy()
    assert np.array_equal(host(y), want, equal_nan=True)


def test_many_short_rows(sess):
    rows, K = 70001, 33
    x = torch.randn((rows, K), generator=torch.Generator().manual_seed(1)).to("cuda")
    codes, scales = torch.zeros((rows, 32), dtype=torch.uint8, device="cuda"), torch.zeros((rows, 2), dtype=torch.uint8, device="cuda")
    y = torch.zeros((rows, K), device="cuda")
    ready()
    ops.mx4_quantize(sess, x, codes, scales)
    ops.mx4_dequantize(sess, codes, scales, y)
    done(sess)
    some = [0, 1, 31, 32, 255, 256, 35000, rows - 2, rows - 1]
    assert np.array_equal(host(y)[some], ref.round_trip(host(x)[some]))


@pytest.mark.parametrize("kind,rows,K,pad", [("f32", 1030, 17000, 0), ("bf16", 2100, 16500, 3)])
def test_results_larger_than_the_caches(sess, kind, rows, K, pad):
    """Values of more than 64 MiB are written with other stores."""
    codes, scales = ref.exact_rows(np.random.default_rng(rows), 37, K)
    pick = np.random.default_rng(1).integers(0, 37, rows)
    y, buf = poisoned(rows, K, kind, K + pad)
    dc, ds = device(codes[pick]), device(scales[pick])
    ready()
    ops.mx4_dequantize(sess, dc, ds, y)
    done(sess)
    want = torch.from_numpy(ref.values(codes, scales, K).astype(np.float32)).to(TYPES[kind]).to("cuda")[torch.from_numpy(pick).to("cuda")]
    assert torch.equal(y, want)
    assert (buf[rows * (K + pad):] == 77).all() and (pad == 0 or (buf[:rows * (K + pad)].view(rows, K + pad)[:, K:] == 77).all())


# ---- products ----------------------------------------------------------------------------


class Layer:
    """Weights of a seeded [N, K] MX4 matrix and its values."""

    def __init__(self, sess, rng, N, K, gate_up=False, make=ref.exact_rows):
        self.codes, self.scales = make(rng, N, K)
        self.values = ref.values(self.codes, self.scales, K)
        self.w = ops.MX4Weights(sess, K, N, self.codes, self.scales, gate_up=gate_up)

    def close(self):
        self.w.close()


def test_the_shapes_take_every_kernel(sess):
    """The lists of sizes below reach every shape of tile, halves of the largest ones, K in parts and both ways to the few-row kernel."""
    taken = {route(sess, M, N, K)[:3] + (route(sess, M, N, K)[3] > 1,) for M, N, K in SHAPES}
    assert {(0, 16, 16, False), (0, 32, 16, False), (0, 32, 32, False), (0, 64, 16, False)} <= taken
    assert {t[:3] for t in taken if t[0]} == {(1, a, b) for a, b in ((256, 256), (128, 128), (64, 128), (128, 64), (64, 64))}
    assert any(t[3] for t in taken)
    big = [(M, N) for M, N, K in SHAPES if route(sess, M, N, K)[:3] == (1, 256, 256)]
    tiles = {-(-M // 256) * -(-N // 256) for M, N in big}
    assert any(t > 256 and 0 < t % 256 <= 128 for t in tiles) # chains with halves behind ...
    assert any(t % 256 > 128 for t in tiles)                   # ... a round of whole tiles
    swiglu = {route(sess, M, F, K, 1)[:3] for M, F, K in SWIGLU} | {route(sess, M, F, H, 1)[:3] for M, H, F in FFN}
    assert {(0, 16, 64), (0, 32, 64), (1, 64, 128), (1, 128, 128), (1, 256, 256)} <= swiglu


def route(sess, M, N, K, swiglu=0):
    out = [C.c_int(0) for _ in range(4)]
    sess.lib.rkh_mx4_route(M, N, K, swiglu, *[C.byref(x) for x in out])
    return tuple(x.value for x in out)


SHAPES = [(1, 1, 1), (1, 32, 32), (1, 33, 31), (1, 129, 500), (2, 64, 513), (3, 200, 4096), (4, 1999, 2050), (5, 100, 128), (16, 4100, 640), (16, 48, 14336),
          (17, 65, 129), (32, 4100, 300), (33, 70, 1100), (61, 1999, 2050), (64, 96, 8192), (65, 31, 33), (65, 300, 8200), (100, 1000, 520), (128, 4096, 512), (129, 257, 1536),
          (130, 11008, 256), (256, 512, 7000), (257, 4096, 96), (300, 12400, 160), (515, 6000, 700), (1025, 2100, 1030), (2048, 4096, 512),
          (20, 17000, 300), (2100, 5900, 700), (4100, 5000, 520)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product_of_exact_rows_bit_for_bit(sess, M, N, K):
    rng = np.random.default_rng(M * 7 + N * 3 + K)
    layer = Layer(sess, rng, N, K)
    a = ref.values(*ref.exact_rows(rng, M, K), K)
    ws = ops.MX4Workspace(sess, M, K, N)
    want = a @ layer.values.T
    for kind, out, pad_a, pad_c in (("f32", "f32", 0, 0), ("bf16", "f16", 3, 5), ("f16", "bf16", 8, 0)):
        x = torch.zeros((M, K + pad_a), dtype=TYPES[kind], device="cuda")[:, :K]
        x.copy_(device(a, kind))
        c, buf = poisoned(M, N, out, N + pad_c)
        ready()
        ws.run(layer.w, x, c)
        done(sess)
        assert np.array_equal(host(c), torch.from_numpy(want).to(TYPES[out]).double().numpy()), (kind, out, route(sess, M, N, K))
        assert untouched(buf, M, N, N + pad_c)
    ws.close()
    layer.close()


def ordinary(rng, rows, K):
    x = rng.standard_normal((rows, K)) * 0.02
    return ref.quantize(x)


@pytest.mark.parametrize("M,N,K", [(1, 512, 4096), (16, 300, 2050), (48, 256, 1000), (200, 384, 4096), (700, 2048, 1030)])
def test_product_of_ordinary_rows_within_fp32_sums(sess, M, N, K):
    """Off by at most K 2^-24 of the sum of magnitudes (K roundings of partial sums) and half a step of the result."""
    rng = np.random.default_rng(M + N + K)
    layer = Layer(sess, rng, N, K, make=ordinary)
    x = rng.standard_normal((M, K)) * np.where(rng.random((M, K)) < 0.005, 20, 1)
    d = device(x, "f32")
    a = ref.round_trip(host(d))
    ws = ops.MX4Workspace(sess, M, K, N)
    want, size = a @ layer.values.T, np.abs(a) @ np.abs(layer.values).T
    for out in ("f32", "f16", "bf16"):
        c = torch.zeros((M, N), dtype=TYPES[out], device="cuda")
        ready()
        ws.run(layer.w, d, c)
        done(sess)
        bound = K * 2.0 ** -24 * size
        far = np.abs(host(c) - want) - bound - HALF_STEP[out] * (np.abs(want) + bound) - (2.0 ** -25 if out == "f16" else 0)
        assert far.max() <= 0, (out, far.max())
    ws.close()
    layer.close()


@pytest.mark.parametrize("M,N,K", [(2, 100, 700), (20, 100, 700), (200, 200, 700)])
def test_nan_stays_in_its_row_and_its_column(sess, M, N, K):
    rng = np.random.default_rng(M)
    codes, scales = ref.exact_rows(rng, N, K)
    scales[N // 2, 3] = 255
    w = ops.MX4Weights(sess, K, N, codes, scales)
    a = ref.values(*ref.exact_rows(rng, M, K), K)
    a[M // 2, K - 1] = np.inf
    ws, x, c = ops.MX4Workspace(sess, M, K, N), device(a, "f32"), torch.zeros((M, N), device="cuda")
    ready()
    ws.run(w, x, c)
    done(sess)
    bad = np.zeros((M, N), bool)
    bad[M // 2] = True
    bad[:, N // 2] = True
    got = host(c)
    assert np.array_equal(np.isnan(got), bad)
    a[M // 2] = 0
    scales[N // 2, 3] = 127
    assert np.array_equal(got[~bad], (a @ ref.values(codes, scales, K).T)[~bad])
    ws.close()
    w.close()


def test_rows_behind_the_last_one_may_hold_anything(sess):
    """A workspace that staged more rows before, NaN among them: fewer rows do not see them."""
    rng = np.random.default_rng(8)
    K, N = 640, 200
    layer = Layer(sess, rng, N, K)
    ws = ops.MX4Workspace(sess, 300, K, N)
    full = torch.full((300, K), float("nan"), device="cuda")
    trash = torch.zeros((300, N), device="cuda")
    for M in (9, 20, 70, 140):
        a = ref.values(*ref.exact_rows(rng, M, K), K)
        x, c = device(a, "f32"), torch.zeros((M, N), device="cuda")
        ready()
        ws.run(layer.w, full, trash)
        ws.run(layer.w, x, c)
        done(sess)
        assert np.array_equal(host(c), a @ layer.values.T), M
        assert np.isnan(host(trash)).all()
    ws.close()
    layer.close()


def test_staged_rows_serve_several_weights(sess):
    rng = np.random.default_rng(5)
    K, rows = 1100, 37
    layers = [Layer(sess, rng, N, K) for N in (512, 64, 200)]
    ws = ops.MX4Workspace(sess, 64, K, 512)
    a = ref.values(*ref.exact_rows(rng, rows, K), K)
    x = device(a, "bf16")
    outs = [torch.zeros((rows, layer.w.N), device="cuda") for layer in layers]
    ready()
    ws.stage(x)
    for layer, c in zip(layers, outs):
        ws.run_staged(layer.w, c)
    done(sess)
    for layer, c in zip(layers, outs):
        assert np.array_equal(host(c), a @ layer.values.T)
    for layer in layers:
        layer.close()
    ws.close()


def test_weights_from_device_arrays_that_quantize_wrote(sess):
    rng = np.random.default_rng(6)
    N, K, M = 130, 333, 40
    x = device(rng.standard_normal((N, K)), "f32")
    codes, scales = torch.zeros((N, 11 * 16), dtype=torch.uint8, device="cuda"), torch.zeros((N, 11), dtype=torch.uint8, device="cuda")
    ready()
    ops.mx4_quantize(sess, x, codes, scales)
    w = ops.MX4Weights.from_device(sess, K, N, codes.data_ptr(), scales.data_ptr())
    config, size = capi.MX4WeightConfig(), C.c_uint64(0)
    assert sess.lib.rk_npu_mx4_weights_query(w.h, C.byref(config), C.byref(size)) == 0
    assert (config.K, config.N, config.gate_up) == (K, N, 0) and size.value >= N * 11 * 17
    a = np.zeros((M, K))
    a[np.arange(M), np.arange(M) * 8] = 1.0 # one-hot rows: the products are the weights' values
    ws, c = ops.MX4Workspace(sess, M, K, N), torch.zeros((M, N), device="cuda")
    d = device(a, "f32")
    ready()
    ws.run(w, d, c)
    done(sess)
    assert np.array_equal(host(c), ref.round_trip(host(x))[:, np.arange(M) * 8].T)
    ws.close()
    w.close()


# ---- SwiGLU and the FFN --------------------------------------------------------------------


def swiglu_bound(gate, up, K, a, g_values, u_values):
    """How far fp32 sums, the exponential, the reciprocal (together below 2^-20 relative) and the products may take silu(gate) * up."""
    eg = K * 2.0 ** -24 * (np.abs(a) @ np.abs(g_values).T)
    eu = K * 2.0 ** -24 * (np.abs(a) @ np.abs(u_values).T)
    s = np.abs(ref.silu(gate))
    return 1.1 * eg * (np.abs(up) + eu) + s * eu + 2.0 ** -19 * s * np.abs(up) + 1e-30


SWIGLU = [(1, 64, 96), (1, 33, 512), (3, 300, 4100), (16, 500, 640), (31, 70, 1000), (33, 96, 300), (100, 350, 1500), (300, 1000, 520), (200, 7000, 200),
          (500, 14300, 130)]


@pytest.mark.parametrize("M,F,K", SWIGLU)
def test_swiglu(sess, M, F, K):
    rng = np.random.default_rng(M + F + K)
    layer = Layer(sess, rng, 2 * F, K, gate_up=True, make=ordinary)
    d = device(rng.standard_normal((M, K)), "f32")
    a = ref.round_trip(host(d))
    g, u = layer.values[:F], layer.values[F:]
    gate, up = a @ g.T, a @ u.T
    want, bound = ref.silu(gate) * up, swiglu_bound(gate, up, K, a, g, u)
    ws = ops.MX4Workspace(sess, M, K, 2 * F)
    for out, pad in (("f32", 0), ("bf16", 3), ("f16", 0)):
        c, buf = poisoned(M, F, out, F + pad)
        ready()
        ws.run_swiglu(layer.w, d, c)
        done(sess)
        far = np.abs(host(c) - want) - bound - HALF_STEP[out] * (np.abs(want) + bound) - (2.0 ** -25 if out == "f16" else 0)
        assert far.max() <= 0, (out, far.max(), route(sess, M, F, K, 1))
        assert untouched(buf, M, F, F + pad)
    ws.close()
    layer.close()


@pytest.mark.parametrize("M", [1, 20, 70, 300])
def test_swiglu_of_far_gates(sess, M):
    """One-hot rows: the sums are single products, exact, over the whole range of the exponential.  16 roundings or ulps around it."""
    K = F = 512
    rng = np.random.default_rng(M)
    gate = np.zeros((F, K))
    up = np.zeros((F, K))
    at = np.arange(F)
    gate[at, at] = np.tile([0, 0.5, -0.5, 1, -1.5, 4, -6, 12, -24, 48, -64, 96, -96, 128, -192, 1024], F // 16)
    up[at, at] = rng.choice([1.0, -2.0, 0.5], F)
    w = ops.MX4Weights(sess, K, 2 * F, *ref.quantize(np.concatenate([gate, up])), gate_up=True)
    x = np.zeros((M, K))
    pick = rng.integers(0, K, M)
    x[np.arange(M), pick] = 1.0
    ws, d, c = ops.MX4Workspace(sess, M, K, 2 * F), device(x, "f32"), torch.zeros((M, F), device="cuda")
    ready()
    ws.run_swiglu(w, d, c)
    done(sess)
    with np.errstate(over="ignore"):
        want = ref.silu(x @ gate.T) * (x @ up.T)
    assert (np.abs(host(c) - want) <= 16 * 2.0 ** -24 * np.abs(want) + 1e-36).all()
    ws.close()
    w.close()


FFN = [(1, 512, 700), (4, 96, 64), (13, 300, 333), (32, 640, 1000), (40, 130, 257), (150, 512, 900), (300, 1024, 1600), (500, 130, 14300)]


@pytest.mark.parametrize("M,H,F", FFN)
def test_ffn_is_its_two_calls_bit_for_bit(sess, M, H, F):
    """The middle that the FFN keeps as MX4 rows is the one that run_swiglu gives in fp32 and run quantizes again."""
    rng = np.random.default_rng(M + H + F)
    gu, dn = Layer(sess, rng, 2 * F, H, gate_up=True, make=ordinary), Layer(sess, rng, H, F, make=ordinary)
    gws, dws = ops.MX4Workspace(sess, M, H, 2 * F), ops.MX4Workspace(sess, M, F, H)
    x = device(rng.standard_normal((M, H)), "bf16")
    middle, two, one = (torch.zeros((M, n), device="cuda") for n in (F, H, H))
    ready()
    # (blocks of the middle beyond F would show: both workspaces are used for something else first)
    full, trash = torch.ones((M, F), device="cuda"), torch.zeros((M, H), device="cuda")
    ready()
    dws.run(dn.w, full, trash)
    ops.mx4_ffn(gws, gu.w, dws, dn.w, x, one)
    gws.run_swiglu(gu.w, x, middle)
    dws.run(dn.w, middle, two)
    done(sess)
    assert np.array_equal(host(one), host(two))
    assert np.isfinite(host(one)).all() and np.abs(host(one)).max() > 0
    want = ref.round_trip(host(middle)) @ dn.values.T
    size = np.abs(ref.round_trip(host(middle))) @ np.abs(dn.values).T
    assert (np.abs(host(two) - want) <= F * 2.0 ** -24 * size + 2.0 ** -24 * np.abs(want)).all()
    for x in (gws, dws, gu, dn):
        x.close()


@pytest.mark.parametrize("M,H,F,kind,gate,after", [(1, 512, 700, "bf16", "channel", True), (5, 333, 260, "f32", "full", False), (33, 640, 300, "f16", "none", True),
                                                   (200, 512, 1000, "bf16", "full", True)])
def test_ffn_block_is_its_calls_bit_for_bit(sess, M, H, F, kind, gate, after):
    """Norm, SwiGLU product, down product and the norms behind it as separate public calls give the block's bits."""
    rng = np.random.default_rng(M + H + F)
    gu, dn = Layer(sess, rng, 2 * F, H, gate_up=True, make=ordinary), Layer(sess, rng, H, F, make=ordinary)
    gws, dws = ops.MX4Workspace(sess, M, H, 2 * F), ops.MX4Workspace(sess, M, F, H)
    stream = device(rng.standard_normal((M, H)), kind)
    before, behind, following = (device(1 + 0.1 * rng.standard_normal(H), "f32") for _ in range(3))
    g = {"none": None, "channel": device(rng.random(H), "bf16"), "full": device(rng.random((M, H)), "bf16")}[gate]
    common = dict(after=behind if after else None, gate=g, residual_scale=0.75, branch_scale=0.5)
    branch, middle = torch.zeros((M, H), device="cuda"), torch.zeros((M, F), device="cuda")
    out = [(torch.zeros_like(stream), torch.zeros((M, H), device="cuda")) for _ in range(3)]
    in_place = stream.clone()
    ready()
    ops.mx4_ffn_block(gws, gu.w, dws, dn.w, stream, branch, weight=before, next_weight=following, stream_out=out[0][0], y=out[0][1], **common)
    done(sess)
    first = host(branch).copy()
    ops.block_norm(sess, stream, weight=before, staged=gws)
    gws.run_staged(gu.w, middle)
    dws.run(dn.w, middle, branch)
    ops.block_norm(sess, stream, branch, weight=following, stream_out=out[1][0], y=out[1][1], **common)
    done(sess)
    assert np.array_equal(host(branch), first)
    ops.mx4_ffn_block(gws, gu.w, dws, dn.w, in_place, branch, weight=before, stream_out=in_place, **common)
    done(sess)
    assert np.array_equal(host(out[0][0]), host(out[1][0])) and np.array_equal(host(out[0][1]), host(out[1][1]))
    assert np.array_equal(host(in_place), host(out[0][0]))
    assert np.isfinite(host(in_place)).all()
    for x in (gws, dws, gu, dn):
        x.close()


# ---- captured, refused, empty ---------------------------------------------------------------


@pytest.mark.parametrize("M", [1, 40, 200])
def test_captured_block_replays_what_the_eager_call_gives(sess, M):
    """Replays between eager calls on other rows and on the same workspaces."""
    rng = np.random.default_rng(M)
    H, F = 512, 600
    gu, dn = Layer(sess, rng, 2 * F, H, gate_up=True, make=ordinary), Layer(sess, rng, H, F, make=ordinary)
    gws, dws = ops.MX4Workspace(sess, M, H, 2 * F), ops.MX4Workspace(sess, M, F, H)
    inputs = [device(rng.standard_normal((M, H)), "bf16") for _ in range(4)]
    x, got, eager = inputs[0].clone(), torch.zeros((M, H), dtype=torch.bfloat16, device="cuda"), torch.zeros((M, H), dtype=torch.bfloat16, device="cuda")
    branch = torch.zeros((M, H), device="cuda")
    call = lambda source, to: ops.mx4_ffn_block(gws, gu.w, dws, dn.w, source, branch, stream_out=to)  # noqa: E731
    ready()
    call(x, got)
    done(sess)
    assert sess.lib.rk_npu_hip_capture_begin(sess.ctx) == 0
    call(x, got)
    graph = sess.lib.rk_npu_hip_capture_end(sess.ctx)
    assert graph
    for source in inputs + inputs[:2]:
        x.copy_(source)
        got.zero_()
        ready()
        assert sess.lib.rk_npu_hip_graph_launch(sess.ctx, graph) == 0
        call(source, eager)
        done(sess)
        assert np.array_equal(host(got), host(eager)) and np.abs(host(got)).max() > 0
    sess.lib.rk_npu_hip_graph_free(graph)
    for h in (gws, dws, gu, dn):
        h.close()


def test_two_captured_graphs_share_workspaces(sess):
    """Two graphs on the same workspaces, replayed in turn with eager calls between them: each stages its own rows."""
    rng = np.random.default_rng(4)
    M, H, N = 70, 640, 200
    layers = [Layer(sess, rng, N, H, make=ordinary) for _ in range(2)]
    ws = ops.MX4Workspace(sess, M, H, N)
    xs = [device(rng.standard_normal((M, H)), "f16") for _ in range(2)]
    outs = [torch.zeros((M, N), device="cuda") for _ in range(4)]

    def call(k, to):
        ws.stage(xs[k])
        ws.run_staged(layers[k].w, to)
    ready()
    graphs = []
    for k in range(2):
        call(k, outs[2 + k])
        done(sess)
        assert sess.lib.rk_npu_hip_capture_begin(sess.ctx) == 0
        call(k, outs[k])
        graphs.append(sess.lib.rk_npu_hip_capture_end(sess.ctx))
        assert graphs[-1]
    for k in (0, 1, 1, 0, 1, 0, 0):
        outs[k].zero_()
        ready()
        assert sess.lib.rk_npu_hip_graph_launch(sess.ctx, graphs[k]) == 0
        call(1 - k, outs[3 - k])
        done(sess)
        assert np.array_equal(host(outs[k]), host(outs[2 + k])) and np.abs(host(outs[k])).max() > 0
    for graph in graphs:
        sess.lib.rk_npu_hip_graph_free(graph)
    for h in layers + [ws]:
        h.close()


def test_offsets_beyond_32_bits(sess):
    """More than 2^32 values in a quantization and in a product's result: the last rows are right, and reading back finds them."""
    rng = np.random.default_rng(9)
    rows, K = 140000, 32768
    last = device(rng.standard_normal((3, K)), "bf16")
    x = torch.zeros((rows, K), dtype=torch.bfloat16, device="cuda")
    x[-3:] = last
    codes, scales = torch.full((rows, K // 2), 0x11, dtype=torch.uint8, device="cuda"), torch.zeros((rows, K // 32), dtype=torch.uint8, device="cuda")
    ready()
    ops.mx4_quantize(sess, x, codes, scales)
    done(sess)
    x[-3:] = 0
    ready()
    ops.mx4_dequantize(sess, codes, scales, x)
    done(sess)
    assert np.array_equal(host(x[-3:]), ref.round_trip(host(last)))
    assert not codes[:-3].any() and not x[:-3].any()
    del x, codes, scales
    M, N = 140000, 32000
    layer = Layer(sess, rng, N, 32)
    a = ref.values(*ref.exact_rows(rng, 64, 32), 32)
    d = device(np.tile(a, (-(-M // 64), 1))[:M], "bf16")
    ws, c = ops.MX4Workspace(sess, M, 32, N), torch.full((M, N), 77.0, dtype=torch.bfloat16, device="cuda")
    ready()
    ws.run(layer.w, d, c)
    done(sess)
    want = torch.from_numpy(a @ layer.values.T).to(torch.bfloat16).to("cuda")
    for at in (0, 67072, 134208, M - 64):
        assert torch.equal(c[at:at + 64], want.roll(-(at % 64), 0)), at
    ws.close()
    layer.close()


def test_zero_rows_write_nothing(sess):
    nothing = torch.zeros((0, 96), device="cuda")
    none = torch.zeros((0, 48), dtype=torch.uint8, device="cuda"), torch.zeros((0, 3), dtype=torch.uint8, device="cuda")
    ops.mx4_quantize(sess, nothing, *none)
    ops.mx4_dequantize(sess, *none, nothing)
    ops.block_norm(sess, nothing, y=nothing.clone())
    rng = np.random.default_rng(1)
    layer = Layer(sess, rng, 64, 96)
    ws = ops.MX4Workspace(sess, 8, 96, 64)
    x, c = torch.ones((1, 96), device="cuda"), torch.full((1, 64), 5.0, device="cuda")
    p, q = C.c_void_p(x.data_ptr()), C.c_void_p(c.data_ptr())
    ready()
    lib = sess.lib
    assert lib.rk_npu_mx4_run_device(ws.h, layer.w.h, 0, 0, p, 96, 0, q, 64) == 0
    assert lib.rk_npu_mx4_quantize_device(sess.ctx, 0, 0, 96, p, 96, q, q) == 0
    assert lib.rk_npu_mx4_dequantize_device(sess.ctx, 0, 0, 96, p, p, q, 96) == 0
    assert lib.rk_npu_mx4_stage_device(ws.h, 0, 0, p, 96) == 0
    assert lib.rk_npu_mx4_run_staged_device(ws.h, layer.w.h, 0, q, 64) == capi.RK_NPU_ERR_PARAM
    done(sess)
    assert (host(c) == 5).all()
    ws.close()
    layer.close()


def test_refusals(sess):
    rng = np.random.default_rng(2)
    K, N = 96, 64
    layer, pair = Layer(sess, rng, N, K), Layer(sess, rng, N, K, gate_up=True)
    ws, small = ops.MX4Workspace(sess, 8, K, N), ops.MX4Workspace(sess, 8, K, N - 1)
    x, c = torch.ones((8, 128), device="cuda"), torch.full((8, 128), 5.0, device="cuda")
    ready()
    lib, bad = sess.lib, capi.RK_NPU_ERR_PARAM
    p, q = x.data_ptr(), c.data_ptr()
    run = lambda ws=ws, w=layer.w, rows=4, at=0, a=p, lda=128, ct=0, out=q, ldc=128: lib.rk_npu_mx4_run_device(ws.h, w.h, rows, at, a, lda, ct, out, ldc)  # noqa: E731
    assert run() == 0
    done(sess)
    for wrong in (dict(rows=-1), dict(rows=9), dict(at=3), dict(at=-1), dict(ct=3), dict(a=None), dict(out=None), dict(lda=K - 1), dict(ldc=N - 1), dict(a=p + 2),
                  dict(out=q + 1), dict(at=1, a=p + 1), dict(w=pair.w), dict(ws=small), dict(out=p), dict(out=p + 4 * 3 * 128), dict(a=q - 4 * 3 * 128 - 4 * 90)):
        assert run(**wrong) == bad, wrong
    assert lib.rk_npu_mx4_run_swiglu_device(ws.h, layer.w.h, 4, 0, p, 128, 0, q, 128) == bad
    assert lib.rk_npu_mx4_run_staged_device(ws.h, layer.w.h, 0, q, 128) == bad # run leaves nothing staged
    assert lib.rk_npu_mx4_run_ffn_device(ws.h, pair.w.h, ws.h, layer.w.h, 4, 0, p, 128, 0, q, 128) == bad
    quant = lambda type=0, rows=2, K=96, x=p, ld=96, codes=q, scales=q + 2048: lib.rk_npu_mx4_quantize_device(sess.ctx, type, rows, K, x, ld, codes, scales)  # noqa: E731
    assert quant() == 0
    for wrong in (dict(type=5), dict(rows=-1), dict(K=0), dict(x=None), dict(ld=95), dict(codes=None), dict(scales=None), dict(codes=p + 100), dict(scales=p), dict(scales=q + 10)):
        assert quant(**wrong) == bad, wrong
    config = capi.MX4WeightConfig(96, 63, 1)
    assert not lib.rk_npu_mx4_weights_create(sess.domain, C.byref(config), layer.codes.ctypes.data, layer.scales.ctypes.data) # half a pair
    for rows, k, n in ((0, 96, 64), (8, 0, 64), (8, 96, 0), (8, 1 << 30, 64)):
        assert not lib.rk_npu_mx4_workspace_create(sess.domain, rows, k, n)
    other = lib.rk_npu_iommu_domain_create(sess.ctx, 3)
    foreign = lib.rk_npu_mx4_workspace_create(other, 8, K, N)
    assert foreign and lib.rk_npu_mx4_run_device(foreign, layer.w.h, 4, 0, p, 128, 0, q, 128) == capi.RK_NPU_ERR_DOMAIN
    lib.rk_npu_mx4_workspace_free(foreign)
    lib.rk_npu_iommu_domain_free(other)
    done(sess)
    for h in (ws, small, layer, pair):
        h.close()


def test_out_of_memory_at_every_allocation(sess):
    rng = np.random.default_rng(3)
    codes, scales = ref.exact_rows(rng, 64, 96)
    config = capi.MX4WeightConfig(96, 64, 0)
    lib = sess.lib
    for n in (1, 2, 3, 4):
        lib.rk_npu_hip_fail_alloc_after(n)
        assert not lib.rk_npu_mx4_weights_create(sess.domain, C.byref(config), codes.ctypes.data, scales.ctypes.data), n
    for n in (1, 2, 3):
        lib.rk_npu_hip_fail_alloc_after(n)
        assert not lib.rk_npu_mx4_workspace_create(sess.domain, 128, 8192, 64), n
    lib.rk_npu_hip_fail_alloc_after(0)
