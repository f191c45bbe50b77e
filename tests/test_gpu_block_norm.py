"""GPU tests of the norms around a block through the C ABI, against the formula in 64 bits.

Tolerance: a sum of D squares in fp32 is off by at most D 2^-24 relative, a root halves that, and the few roundings around it
(mean, root, quotient, factor, weight; gate, scales and the fused add) are 2^-24 each: (D / 2 + 8) 2^-24 of y for each norm
that it goes through, 8 of them for the terms of r.  An output's own rounding adds half a step.
"""
import ctypes as C

import numpy as np
import pytest
import torch

from rknpu2_matmul_open_amd import capi, ops
from tests import mx4_reference as ref
from tests.test_gpu_mx4 import HALF_STEP, TYPES, device, done, host, poisoned, ready, untouched

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def reference(stream, branch, after, gate, a, b, weight, eps):
    """r, y and how far fp32 may be off either."""
    D = stream.shape[1]
    norm = (D / 2 + 8) * U
    r, off = stream, np.zeros_like(stream)
    if branch is not None:
        z = branch if after is None else ref.rms(branch, eps, after)
        z = z if gate is None else z * gate
        r = a * stream + b * z
        off = 8 * U * (np.abs(a * stream) + np.abs(b * z)) + (norm if after is not None else 0) * np.abs(b * z)
    root = np.sqrt((r * r).mean(axis=1, keepdims=True) + eps)
    y = r / root * (1 if weight is None else weight)
    # r's own error: in the value, and in the root
    grown = (off + np.abs(r) * np.sqrt((off * off).mean(axis=1, keepdims=True)) / root) / root * (1 if weight is None else np.abs(weight))
    return r, off, y, norm * np.abs(y) + 1.01 * grown


def check(got, want, off, kind, what):
    far = np.abs(host(got) - want) - off - HALF_STEP[kind] * (np.abs(want) + off) - (2.0 ** -25 if kind == "f16" else 1e-38)
    assert far.max() <= 0, (what, far.max())


CASES = [(1, 1, "f32", "f32", "f32", True, "full"), (3, 7, "f32", "bf16", "f16", True, "channel"), (5, 8, "bf16", "bf16", "bf16", False, "none"),
         (2, 255, "f16", "f16", "f32", True, "none"), (4, 2048, "f32", "bf16", "bf16", True, "full"), (3, 2049, "bf16", "f32", "f32", True, "channel"),
         (130, 4096, "f32", "f32", "f32", False, "full"), (2, 5000, "f16", "bf16", "f16", True, "full"), (2, 16384, "f32", "f32", "f32", True, "channel"),
         (3, 16385, "f32", "bf16", "f32", True, "full"), (2, 40001, "bf16", "bf16", "f32", False, "channel"), (1000, 96, "bf16", "f16", "f32", True, "full")]


@pytest.mark.parametrize("rows,D,stream_kind,branch_kind,y_kind,after,gate", CASES)
def test_against_the_formula(sess, rows, D, stream_kind, branch_kind, y_kind, after, gate):
    rng = np.random.default_rng(rows + D)
    pad = 3
    stream = torch.zeros((rows, D + pad), dtype=TYPES[stream_kind], device="cuda")[:, :D]
    stream.copy_(device(rng.standard_normal((rows, D)) * 3, stream_kind))
    branch = torch.zeros((rows, D + 1), dtype=TYPES[branch_kind], device="cuda")[:, :D]
    branch.copy_(device(rng.standard_normal((rows, D)) * np.exp2(rng.integers(-6, 6, (rows, 1))), branch_kind))
    g = {"none": None, "channel": device(rng.standard_normal(D), "bf16"), "full": device(rng.standard_normal((rows, D)), "f16")}[gate]
    weight, behind = device(1 + 0.2 * rng.standard_normal(D), "f32"), device(1 + 0.2 * rng.standard_normal(D), "f32")
    out, out_buf = poisoned(rows, D, stream_kind, D + 2)
    y, y_buf = poisoned(rows, D, y_kind, D + 5)
    ready()
    ops.block_norm(sess, stream, branch, after=behind if after else None, gate=g, residual_scale=0.75, branch_scale=-1.5, weight=weight, eps=1e-5, stream_out=out, y=y)
    done(sess)
    r, r_off, want, y_off = reference(host(stream), host(branch), host(behind) if after else None, None if g is None else host(g), 0.75, -1.5, host(weight),
                                      float(np.float32(1e-5)))
    check(out, r, r_off, stream_kind, "stream")
    check(y, want, y_off, y_kind, "y")
    assert untouched(out_buf, rows, D, D + 2) and untouched(y_buf, rows, D, D + 5)


@pytest.mark.parametrize("D", [64, 3000, 20000])
def test_parts_left_out(sess, D):
    rng = np.random.default_rng(D)
    stream, branch = device(rng.standard_normal((3, D)), "f32"), device(rng.standard_normal((3, D)), "f32")
    y, out = torch.zeros((3, D), device="cuda"), torch.zeros((3, D), device="cuda")
    ready()
    ops.block_norm(sess, stream, y=y)                                # a norm alone, without weight
    done(sess)
    _, _, want, off = reference(host(stream), None, None, None, 1, 1, None, 1e-6)
    check(y, want, off, "f32", "norm alone")
    ready()
    ops.block_norm(sess, stream, branch, residual_scale=2.0, branch_scale=0.5, stream_out=out) # a scaled add alone: exact but for one rounding
    done(sess)
    assert (np.abs(host(out) - (2 * host(stream) + 0.5 * host(branch))) <= U * np.abs(2 * host(stream) + 0.5 * host(branch))).all()
    ready()
    ops.block_norm(sess, stream, residual_scale=2.0, stream_out=out) # no branch: the stream as it is
    done(sess)
    assert np.array_equal(host(out), host(stream))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("D", [200, 4096, 17000])
def test_in_place_gives_the_same_bits(sess, D, kind):
    rng = np.random.default_rng(D)
    stream, branch = device(rng.standard_normal((5, D)), kind), device(rng.standard_normal((5, D)), "bf16")
    behind = device(rng.random(D), "f32")
    apart, y, y2 = torch.zeros_like(stream), torch.zeros((5, D), device="cuda"), torch.zeros((5, D), device="cuda")
    ready()
    ops.block_norm(sess, stream, branch, after=behind, stream_out=apart, y=y)
    ops.block_norm(sess, stream, branch, after=behind, stream_out=stream, y=y2)
    done(sess)
    assert np.array_equal(host(apart), host(stream)) and np.array_equal(host(y), host(y2))


def test_rows_of_zeros_infinities_and_nan(sess):
    D = 300
    x = np.ones((5, D))
    x[0] = 0
    x[1, 7] = np.inf
    x[2, 299] = np.nan
    x[3] = 1e30                 # squares beyond fp32
    stream, y = device(x, "f32"), torch.full((5, D), 7.0, device="cuda")
    ready()
    ops.block_norm(sess, stream, y=y)
    done(sess)
    got = host(y)
    assert (got[0] == 0).all() and np.isnan(got[1, 7]) and np.isnan(got[2]).all()
    assert (got[3] == 0).all()  # the factor of an infinite mean square is 0
    assert (np.abs(got[4] - 1 / np.sqrt(1 + 1e-6)) < 1e-6).all()


@pytest.mark.parametrize("rows,D", [(1, 32), (3, 100), (20, 640), (5, 4097), (2, 16500)])
def test_staged_rows_are_the_quantized_y(sess, rows, D):
    """One-hot weights give the staged values back: those of y in fp32, quantized."""
    rng = np.random.default_rng(D)
    stream, weight = device(rng.standard_normal((rows, D)), "bf16"), device(1 + 0.1 * rng.standard_normal(D), "f32")
    ws = ops.MX4Workspace(sess, rows, D, 64)
    picks = rng.permutation(D)[:min(D, 64)]
    one_hot = np.zeros((len(picks), D))
    one_hot[np.arange(len(picks)), picks] = 1
    w = ops.MX4Weights(sess, D, len(picks), *ref.quantize(one_hot))
    y, c = torch.zeros((rows, D), device="cuda"), torch.zeros((rows, len(picks)), device="cuda")
    ready()
    ops.block_norm(sess, stream, weight=weight, y=y, staged=ws)
    ws.run_staged(w, c)
    done(sess)
    assert np.array_equal(host(c), ref.round_trip(host(y))[:, picks])
    ws.close()
    w.close()


def test_rows_of_more_than_one_launch(sess):
    """A launch holds 2^31 threads at most: rows before and behind that line are what they are on their own."""
    rows, D = (1 << 25) + 9, 2
    x = torch.full((rows, D), 3.0, dtype=torch.float16, device="cuda")
    near = slice((1 << 25) - 5, rows)
    x[near] = device(np.random.default_rng(2).standard_normal((14, D)), "f16")
    y, alone = torch.zeros_like(x), torch.zeros((14, D), dtype=torch.float16, device="cuda")
    ready()
    ops.block_norm(sess, x, y=y)
    ops.block_norm(sess, x[near], y=alone)
    done(sess)
    assert torch.equal(y[near], alone) and alone.abs().min() > 0
    assert (y[:near.start] == 1).all()


def test_refusals(sess):
    rows, D = 4, 64
    buf = torch.ones(8 * rows * D, device="cuda")
    at = lambda i: buf.data_ptr() + 4 * rows * D * i  # noqa: E731
    ws = ops.MX4Workspace(sess, 3, D, 32)
    ready()

    def call(**changed):
        a = capi.BlockNormArgs()
        sess.lib.rk_npu_block_norm_args_init(C.byref(a), rows, D)
        a.residual, a.branch, a.gate, a.residual_out, a.y = at(0), at(1), at(2), at(3), at(4)
        a.residual_ld = a.branch_ld = a.gate_ld = a.residual_out_ld = a.y_ld = D
        for k, v in changed.items():
            setattr(a, k, v)
        return sess.lib.rk_npu_block_norm_device(sess.ctx, C.byref(a))
    assert call() == 0
    assert call(residual_out=at(0)) == 0 and call(rows=0) == 0 and call(gate_ld=0) == 0
    done(sess)
    for wrong in (dict(struct_size=8), dict(rows=-1), dict(D=0), dict(residual=None), dict(residual_type=7), dict(branch_type=-1), dict(gate_type=3), dict(y_type=9),
                  dict(residual_ld=D - 1), dict(branch_ld=1), dict(gate_ld=D - 1), dict(y_ld=0), dict(residual_out_ld=2), dict(eps=-1.0), dict(eps=float("nan")),
                  dict(y=None, residual_out=None), dict(y=at(0)), dict(y=at(1)), dict(y=at(3)), dict(residual_out=at(1) + 4), dict(residual_out=at(0) + 4),
                  dict(residual_out=at(2)), dict(branch=None), dict(branch=None, gate=None, branch_weight=at(5)), dict(weight=at(5) + 2), dict(weight=at(4)),
                  dict(residual=at(0) + 1), dict(staged=ws.h)):
        assert call(**wrong) == capi.RK_NPU_ERR_PARAM, wrong
    assert sess.lib.rk_npu_block_norm_device(sess.ctx, None) == capi.RK_NPU_ERR_PARAM
    ws.close()
