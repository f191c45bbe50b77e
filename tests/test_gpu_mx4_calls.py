"""GPU tests of MX4 and block norm calls that a program may make of them beyond the plain ones: operands that are slices of one buffer.

Products of exact_rows are compared bit for bit; the other calls with the same call on buffers of their own.
"""
import ctypes as C

import numpy as np
import pytest
import torch

from rknpu2_matmul_open_amd import capi, ops
from tests import mx4_reference as ref
from tests.test_gpu_mx4 import Layer, TYPES, device, done, host, ordinary, ready

pytestmark = pytest.mark.gpu


# ---- column slices of one buffer ---------------------------------------------------------


def halves(rows, left, right, kind="f32", gap=0):
    """Two slices of one buffer of 77s, of `left` and `right` columns, and the buffer."""
    buf = torch.full((rows, left + gap + right + 3), 77.0, dtype=TYPES[kind], device="cuda")
    return buf[:, :left], buf[:, left + gap:left + gap + right], buf


@pytest.mark.parametrize("M", [1, 3, 20, 200, 1100])
@pytest.mark.parametrize("swap", [False, True])
def test_product_between_the_slices_of_a_buffer(sess, M, swap):
    """Rows and result as column slices of one buffer, either one first."""
    rng = np.random.default_rng(M)
    K, N = 520, 100
    layer = Layer(sess, rng, N, K)
    a = ref.values(*ref.exact_rows(rng, M, K), K)
    ws = ops.MX4Workspace(sess, M, K, N)
    first, second, buf = halves(M, *((N, K) if swap else (K, N)))
    x, c = (second, first) if swap else (first, second)
    x.copy_(device(a, "f32"))
    ready()
    ws.run(layer.w, x, c)
    done(sess)
    assert np.array_equal(host(c), a @ layer.values.T) and np.array_equal(host(x), a)
    assert (host(buf)[:, K + N:] == 77).all()
    # a result of another type in the same buffer: its pitch in bytes is the rows' own
    as_half = buf.view(torch.float16)
    at = 0 if swap else 2 * K
    half = as_half[:, at:at + N]
    ready()
    ws.run(layer.w, x, half)
    done(sess)
    assert np.array_equal(host(half), torch.from_numpy(a @ layer.values.T).half().double().numpy()) and np.array_equal(host(x), a)
    ws.close()
    layer.close()


@pytest.mark.parametrize("M,H,F", [(1, 64, 96), (5, 333, 260), (200, 512, 1000)])
def test_ffn_calls_between_the_slices_of_a_buffer(sess, M, H, F):
    rng = np.random.default_rng(M + H)
    gu, dn = Layer(sess, rng, 2 * F, H, gate_up=True, make=ordinary), Layer(sess, rng, H, F, make=ordinary)
    gws, dws = ops.MX4Workspace(sess, M, H, 2 * F), ops.MX4Workspace(sess, M, F, H)
    value = device(rng.standard_normal((M, H)), "f32")
    x, c, _ = halves(M, H, H)
    x.copy_(value)
    want, middle, want_middle = torch.zeros((M, H), device="cuda"), halves(M, H, F), torch.zeros((M, F), device="cuda")
    middle[0].copy_(value)
    branch, stream_out, _ = halves(M, H, H, gap=2)
    y, want_out, want_y = torch.zeros((M, H), device="cuda"), torch.zeros((M, H), device="cuda"), torch.zeros((M, H), device="cuda")
    ready()
    ops.mx4_ffn(gws, gu.w, dws, dn.w, value, want)
    ops.mx4_ffn(gws, gu.w, dws, dn.w, x, c)
    gws.run_swiglu(gu.w, value, want_middle)
    gws.run_swiglu(gu.w, middle[0], middle[1])
    done(sess)
    assert torch.equal(c, want) and torch.equal(x, value) and torch.equal(middle[1], want_middle) and want.abs().max() > 0
    ops.mx4_ffn_block(gws, gu.w, dws, dn.w, value, want, stream_out=want_out, y=want_y)
    ops.mx4_ffn_block(gws, gu.w, dws, dn.w, value, branch, stream_out=stream_out, y=y)
    done(sess)
    assert torch.equal(branch, want) and torch.equal(stream_out, want_out) and torch.equal(y, want_y)
    for h in (gws, dws, gu, dn):
        h.close()


@pytest.mark.parametrize("rows,D", [(1, 40), (4, 64), (9, 4096), (3, 17000)])
def test_norm_between_the_slices_of_a_buffer(sess, rows, D):
    """Stream, branch, gate and both outputs as slices of one buffer, the stream in place in the second call."""
    rng = np.random.default_rng(D)
    buf = torch.zeros((rows, 5 * D + 1), device="cuda")
    stream, branch, gate, out, y = (buf[:, i * D:(i + 1) * D] for i in range(5))
    buf.copy_(device(rng.standard_normal((rows, 5 * D + 1)), "f32"))
    apart = [t.clone() for t in (stream, branch, gate)]
    want_out, want_y = torch.zeros((rows, D), device="cuda"), torch.zeros((rows, D), device="cuda")
    ready()
    ops.block_norm(sess, apart[0], apart[1], gate=apart[2], residual_scale=0.5, stream_out=want_out, y=want_y)
    ops.block_norm(sess, stream, branch, gate=gate, residual_scale=0.5, stream_out=out, y=y)
    done(sess)
    assert torch.equal(out, want_out) and torch.equal(y, want_y)
    assert all(torch.equal(t, was) for t, was in zip((stream, branch, gate), apart))
    y.zero_()
    ready()
    ops.block_norm(sess, stream, branch, gate=gate, residual_scale=0.5, stream_out=stream, y=y)
    done(sess)
    assert torch.equal(stream, want_out) and torch.equal(y, want_y)


def test_values_read_back_beside_their_codes(sess):
    """A buffer that holds each row's codes and values next to each other is no MX4 matrix, but values between other values' rows are fine."""
    rows, K = 6, 64
    buf = torch.full((rows, 2 * K), 77.0, device="cuda")
    codes, scales = torch.zeros((rows, 32), dtype=torch.uint8, device="cuda"), torch.zeros((rows, 2), dtype=torch.uint8, device="cuda")
    buf[:, K:] = device(np.random.default_rng(3).standard_normal((rows, K)), "f32")
    want = ref.round_trip(host(buf[:, K:]))
    ready()
    ops.mx4_quantize(sess, buf[:, K:], codes, scales)
    ops.mx4_dequantize(sess, codes, scales, buf[:, :K])
    done(sess)
    assert np.array_equal(host(buf[:, :K]), want)


def test_slices_that_share_a_column_are_refused(sess):
    rng = np.random.default_rng(1)
    K, N, M = 96, 64, 4
    layer = Layer(sess, rng, N, K)
    ws = ops.MX4Workspace(sess, M, K, N)
    buf = torch.ones((M + 2, K + N), device="cuda")
    ready()
    for x, c in ((buf[:M, :K], buf[:M, K - 1:K + N - 1]), (buf[:M, N:], buf[:M, 1:N + 1]), (buf[:M, :K], buf[1:M + 1, K - 1:K + N - 1]),
                 (buf[1:M + 1, N:], buf[:M, 1:N + 1])):
        with pytest.raises(ops.RkError) as e:
            ws.run(layer.w, x, c)
        assert e.value.code == capi.RK_NPU_ERR_PARAM
    # rows of two pitches in one range, though no byte is shared
    flat = torch.ones(4096, device="cuda")
    q = flat.data_ptr()
    assert sess.lib.rk_npu_mx4_run_device(ws.h, layer.w.h, 2, 0, C.c_void_p(q), 512, 0, C.c_void_p(q + 4 * 100), 64) == capi.RK_NPU_ERR_PARAM
    a = capi.BlockNormArgs()
    sess.lib.rk_npu_block_norm_args_init(C.byref(a), 3, 64)
    a.residual, a.residual_ld, a.residual_out, a.residual_out_ld, a.y, a.y_ld = q, 200, q + 4 * 64, 200, q + 4 * 127, 200
    assert sess.lib.rk_npu_block_norm_device(sess.ctx, C.byref(a)) == capi.RK_NPU_ERR_PARAM
    a.y = q + 4 * 128
    assert sess.lib.rk_npu_block_norm_device(sess.ctx, C.byref(a)) == 0
    done(sess)
    # a weight of one row in the gap between rows: no output touches it
    a.weight = q + 4 * 192
    a.D = 8
    assert sess.lib.rk_npu_block_norm_device(sess.ctx, C.byref(a)) == 0
    a.weight = q + 4 * 135
    assert sess.lib.rk_npu_block_norm_device(sess.ctx, C.byref(a)) == capi.RK_NPU_ERR_PARAM
    done(sess)
    ws.close()
    layer.close()


# ---- more blocks than one launch has threads for -------------------------------------------
# A launch holds fewer than 2^32 threads.  Rows of one value keep the memory small: 17 bytes each as MX4 rows, 272 as operand blocks.


def room():
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def test_rows_of_more_blocks_than_a_launch_has_threads_for(sess):
    """Quantization and reading back of more than 2^32 blocks: beside every multiple of 2^31, and at the end, rows are what they are."""
    room()
    rows = (1 << 32) + 300
    near = [slice(0, 64)] + [slice((m << 31) - 64, (m << 31) + 64) for m in (1, 2)] + [slice(rows - 64, rows)]
    rng = np.random.default_rng(2)
    x = torch.ones((rows, 1), dtype=torch.float16, device="cuda")
    for at in near:
        x[at] = device(rng.standard_normal((at.stop - at.start, 1)), "f16")
    codes, scales = torch.zeros((rows, 16), dtype=torch.uint8, device="cuda"), torch.zeros((rows, 1), dtype=torch.uint8, device="cuda")
    ready()
    ops.mx4_quantize(sess, x, codes, scales)
    done(sess)
    for at in near:
        want = ref.quantize(host(x[at]))
        assert np.array_equal(codes[at].cpu().numpy(), want[0]) and np.array_equal(scales[at].cpu().numpy(), want[1]), at
    values = [host(x[at]) for at in near]
    x.fill_(7)
    ready()
    ops.mx4_dequantize(sess, codes, scales, x)
    done(sess)
    for at, was in zip(near, values):
        assert np.array_equal(host(x[at]), ref.round_trip(was)), at
    for piece in x.view(-1).split(1 << 30): # the others are ones but for the slices above
        assert int((piece != 1).sum()) <= 4 * 128
    del x, codes, scales, piece
    room()


def test_staged_rows_of_more_blocks_than_a_launch_has_threads_for(sess):
    room()
    rows, w = (1 << 28) + 17, 1.5
    weights = ops.MX4Weights(sess, 1, 1, *ref.quantize(np.array([[w]])))
    ws = ops.MX4Workspace(sess, rows, 1, 1)
    x = (torch.arange(rows, device="cuda") % 7 - 3).to(torch.float16).view(rows, 1) # (each is a code of its block's scale)
    c = torch.full((rows, 1), 77.0, dtype=torch.float16, device="cuda")
    ready()
    ws.run(weights, x, c)
    done(sess)
    assert torch.equal(c, x * w)
    ws.close()
    weights.close()
    del x, c
    room()


def test_weights_of_more_blocks_than_a_launch_has_threads_for(sess):
    room()
    N = (1 << 28) + 64
    codes, scales = torch.zeros((N, 16), dtype=torch.uint8, device="cuda"), torch.full((N, 1), 127, dtype=torch.uint8, device="cuda")
    codes[:, 0] = (torch.arange(N, device="cuda") % 15).to(torch.uint8)
    ready()
    weights = ops.MX4Weights.from_device(sess, 1, N, codes.data_ptr(), scales.data_ptr())
    del scales
    ws = ops.MX4Workspace(sess, 1, 1, N)
    x, c = torch.full((1, 1), 2.0, device="cuda"), torch.full((1, N), 77.0, dtype=torch.float16, device="cuda")
    ready()
    ws.run(weights, x, c)
    done(sess)
    table = torch.from_numpy(2 * ref.SIGNED).half().to("cuda")
    for k in range(0, N, 1 << 26):
        assert torch.equal(c[0, k:k + (1 << 26)], table[codes[k:k + (1 << 26), 0].int()]), k
    ws.close()
    weights.close()
    del codes, c, x
    room()


# ---- empty batches -------------------------------------------------------------------------


def test_batches_of_no_rows_go_through_every_wrapper(sess):
    """What a program does with a batch, done with an empty one: no call fails, and the calls behind it are right."""
    rng = np.random.default_rng(11)
    H, F = 96, 64
    gu, dn, layer = Layer(sess, rng, 2 * F, H, gate_up=True), Layer(sess, rng, H, F), Layer(sess, rng, 50, H)
    gws, dws = ops.MX4Workspace(sess, 8, H, 2 * F), ops.MX4Workspace(sess, 8, F, H)
    empty = lambda n: torch.zeros((0, n), device="cuda")  # noqa: E731
    a = ref.values(*ref.exact_rows(rng, 3, H), H)
    x, c = device(a, "f32"), torch.zeros((3, 50), device="cuda")
    ready()
    with pytest.raises(ValueError):
        gws.run_staged(layer.w, empty(50)) # nothing staged yet
    gws.run(layer.w, empty(H), empty(50))
    gws.run_swiglu(gu.w, empty(H), empty(F))
    ops.mx4_ffn(gws, gu.w, dws, dn.w, empty(H), empty(H))
    ops.mx4_ffn_block(gws, gu.w, dws, dn.w, empty(H), empty(H), stream_out=empty(H))
    with pytest.raises(ValueError):
        gws.run_staged(layer.w, empty(50)) # run leaves nothing staged
    for stage in (lambda rows: gws.stage(rows), lambda rows: ops.block_norm(sess, rows, staged=gws)):
        stage(empty(H))
        gws.run_staged(layer.w, empty(50))
        gws.run_staged(gu.w, empty(F))
        with pytest.raises(ValueError):
            gws.run_staged(layer.w, c)
        stage(x)
        gws.run_staged(layer.w, c)
    gws.stage(x)
    gws.run_staged(layer.w, c)
    done(sess)
    assert np.array_equal(host(c), a @ layer.values.T)
    for h in (gws, dws, gu, dn, layer):
        h.close()


# ---- weights from tensors --------------------------------------------------------------------


def test_weights_from_tensors_on_the_device(sess):
    """The tensors that quantization fills, or their addresses: the same weights.  Tensors too short are refused, not read past their end."""
    rng = np.random.default_rng(12)
    N, K = 70, 333
    x = device(rng.standard_normal((N, K)), "f32")
    codes, scales = torch.zeros((N, 176), dtype=torch.uint8, device="cuda"), torch.zeros((N, 11), dtype=torch.uint8, device="cuda")
    eye = torch.eye(K, device="cuda")
    ready()
    ops.mx4_quantize(sess, x, codes, scales)
    both = [ops.MX4Weights.from_device(sess, K, N, codes, scales), ops.MX4Weights.from_device(sess, K, N, codes.data_ptr(), scales.data_ptr())]
    ws, outs = ops.MX4Workspace(sess, K, K, N), [torch.zeros((K, N), device="cuda") for _ in both]
    ready()
    for w, c in zip(both, outs):
        ws.run(w, eye, c)
    done(sess)
    assert torch.equal(*outs) and np.array_equal(host(outs[0]).T, ref.round_trip(host(x)))
    for bad in ((codes[:, :160], scales), (codes[1:], scales), (codes, scales[:, :10]), (codes.int(), scales), (codes.cpu(), scales)):
        with pytest.raises(ValueError):
            ops.MX4Weights.from_device(sess, K, N, *bad)
    for h in both + [ws]:
        h.close()


# ---- the ends of the norm's range ------------------------------------------------------------


@pytest.mark.parametrize("rows,D", [(1, 512), (4, 4096), (3, 20000)])
def test_sums_of_squares_at_the_end_of_fp32(sess, rows, D):
    """Rows whose sum of squares is just inside fp32 are normed, rows whose sum is just beyond are zero, in both norms."""
    largest = 2.0 ** 64 / np.sqrt(D)  # D of its squares: 2^128
    sign = np.where(np.arange(D) % 3 == 0, -1.0, 1.0)
    inside, beyond = (np.tile(sign * largest * f, (rows, 1)) for f in (0.99, 1.01))
    y, z = torch.full((rows, D), 7.0, device="cuda"), torch.full((rows, D), 7.0, device="cuda")
    for values, want in ((inside, 1.0), (beyond, 0.0)):
        stream = device(values, "f32")
        nothing = torch.zeros_like(stream)
        ones = torch.ones(D, device="cuda")
        ready()
        ops.block_norm(sess, stream, y=y)
        ops.block_norm(sess, nothing, stream, after=ones, stream_out=z)
        done(sess)
        for got in (host(y), host(z)):
            assert (np.abs(got - want * sign) <= (D / 2 + 8) * 2.0 ** -24).all()
        if D == 512:
            ws, w = ops.MX4Workspace(sess, rows, D, D), ops.MX4Weights(sess, D, D, *ref.quantize(np.eye(D)))
            c = torch.full((rows, D), 7.0, device="cuda")
            ready()
            ops.block_norm(sess, stream, staged=ws)
            ws.run_staged(w, c)
            done(sess)
            assert np.array_equal(host(c), ref.round_trip(host(y)))
            ws.close()
            w.close()


# ---- SwiGLU where the quotient is small ------------------------------------------------------


@pytest.mark.parametrize("M", [1, 20, 70, 300])
def test_swiglu_where_the_exponential_is_near_the_end_of_fp32(sess, M):
    """Gates of -79.5 .. -88.5, each an exact sum of products, with up to 2^100 behind them: silu is 1e-33 .. 3e-37, and none of it is lost.  Relative to it
    16 roundings or ulps, as for other gates.  (From -88.73 on exp is beyond fp32, and silu with it.)"""
    K, F = 64, 512
    rng = np.random.default_rng(M)
    gate, up = np.zeros((F, K)), np.zeros((F, K))
    gate[:, 0] = -64
    gate[:, 32] = rng.choice([-16, -24], F)
    gate[:, 33] = rng.choice([0, -2, 2], F)
    up[:, 0] = rng.choice([1.0, 2.0 ** 20, 2.0 ** 60, 2.0 ** 100], F)
    codes, scales = ref.quantize(np.concatenate([gate, up]))
    values = ref.values(codes, scales, K)
    w = ops.MX4Weights(sess, K, 2 * F, codes, scales, gate_up=True)
    x = np.zeros((M, K))
    x[:, 0] = x[:, 32] = 1.0
    x[::2, 33] = 0.25
    x = ref.round_trip(x)
    ws, d, c = ops.MX4Workspace(sess, M, K, 2 * F), device(x, "f32"), torch.zeros((M, F), device="cuda")
    ready()
    ws.run_swiglu(w, d, c)
    done(sess)
    g = x @ values[:F].T
    want = ref.silu(g) * (x @ values[F:].T)
    assert g.min() == -88.5 and g.max() == -79.5 and len(np.unique(g)) == 6 and (np.abs(want) > 2.0 ** -122).all()
    assert (np.abs(host(c) - want) <= 16 * 2.0 ** -24 * np.abs(want)).all()
    ws.close()
    w.close()
