"""GPU tests of the heads' norm and rotation through the C ABI, against the definition in 64 bits (g4_reference).

Off by, relative to a head's largest value after the norm (a rotation moves values between a pair's two):
  the sum of squares: D roundings of positive terms, half of that in its root; root, reciprocal and two products: 4 roundings or ulps of 2^-23;
  the turn: an angle of 2^-25 turns, pi 2^-24 absolute, its sine and cosine 2 ulps, the scale, two products and a sum: 8 times 2^-23;
  positions of 2^31: angles of 64 bits below 2^31 are rounded by 2^-23, here and in the definition, 1 / 2 pi by as much, and the turns by 1.6 2^-23: 5 more;
and half a step of the type.
"""
import ctypes as C

import numpy as np
import pytest
import torch

from rknpu2_matmul_open_amd import capi, ops
from tests import g4_reference as ref
from tests.test_gpu_mx4 import TYPES, device, done, host, ready

pytestmark = pytest.mark.gpu


def bound(want, D, kind, norm=True, far=False):
    top = np.abs(want).max(axis=2, keepdims=True) * 1.4143
    return top * ((D * 2.0 ** -25 + 4 * 2.0 ** -23 if norm else 0) + (13 if far else 8) * 2.0 ** -23) + ref.HALF_STEP[kind] * np.abs(want) * 1.0001 + ref.LEAST[kind]


class Case:
    """Seeded tensors of [rows, heads, D] as `layout` says, and everything else a call takes."""

    def __init__(self, rows, q_heads, k_heads, D, R, kind, norm=True, axes=1, neighbours=False, interleaved=False, weight="both", scale=1.0, eps=1e-6, far=False, seed=0):
        rng = self.rng = np.random.default_rng(rows * 31 + D * 7 + R + seed)
        self.rows, self.D, self.kind, self.norm, self.eps, self.neighbours, self.scale, self.far = rows, D, kind, norm, eps, neighbours, scale, far
        make = lambda heads: device(rng.standard_normal((rows, heads, D)) * np.exp2(rng.integers(-4, 5, (rows, heads, 1))), kind) if heads else None  # noqa: E731
        self.q, self.k = make(q_heads), make(k_heads)
        vector = lambda: device(1 + 0.3 * rng.standard_normal(D)).float()  # noqa: E731
        self.wq, self.wk = (vector() if norm and q_heads and weight in ("both", "q") else None), (vector() if norm and k_heads and weight in ("both", "k") else None)
        pairs = R // 2
        self.inv_freq = device((10000.0 ** (-np.arange(pairs) / max(1, pairs))).astype(np.float32)) if R else None
        top = 2 ** 31 - 1 if far else 4096
        p = rng.integers(-top - 1 if far else 0, top + 1, (axes, rows))
        if far:
            p.reshape(-1)[:2] = (-2 ** 31, 2 ** 31 - 1)[:p.size]
        self.positions = device(p.astype(np.int32)) if R else None
        sections = [pairs // axes + (i < pairs % axes) for i in range(axes)]
        self.pair_axis = ops.pair_axes(sections, interleaved) if R and axes > 1 else None

    def call(self, sess, q, k, q_out=None, k_out=None):
        ready()
        ops.heads_norm_rotate(sess, q, k, q_out, k_out, norm=self.norm, eps=self.eps, q_weight=self.wq, k_weight=self.wk, positions=self.positions, inv_freq=self.inv_freq,
                              pair_axis=self.pair_axis, neighbours=self.neighbours, rotation_scale=self.scale)

    def want(self, x, weight):
        y = host(x)
        if self.norm:
            y = ref.head_norm(y, None if weight is None else host(weight), self.eps)
        if self.inv_freq is not None:
            freq = host(self.inv_freq)
            y = ref.rotate(y, host(self.positions), freq, self.pair_axis or [0] * len(freq), self.neighbours, self.scale)
        return y

    def check(self, got_q, got_k):
        for x, w, got in ((self.q, self.wq, got_q), (self.k, self.wk, got_k)):
            if x is None:
                continue
            want = self.want(x, w)
            far = np.abs(host(got) - want) - bound(want, self.D, self.kind, self.norm, self.far)
            assert far.max() <= 0, (far.max(), np.argwhere(far > 0)[:5])


CASES = [(1, 32, 8, 128, 128, "bf16", {}), (1, 1, 0, 1, 0, "f32", {}), (3, 0, 2, 2, 2, "f16", {}), (5, 3, 3, 7, 4, "f32", {}), (9, 2, 1, 512, 512, "f16", {}), (2, 5, 1, 511, 510, "bf16", {}),
         (4, 2, 2, 512, 6, "f32", {}), (33, 4, 2, 64, 32, "bf16", {}), (33, 4, 2, 64, 32, "bf16", dict(neighbours=True)), (17, 3, 1, 80, 80, "f16", dict(neighbours=True)),
         (17, 3, 1, 90, 60, "f32", dict(neighbours=True)), (20, 2, 2, 96, 16, "f16", dict(norm=False)), (20, 2, 2, 100, 0, "f32", {}), (20, 2, 2, 128, 0, "bf16", {}),
         (50, 4, 2, 128, 128, "bf16", dict(axes=3)), (50, 4, 2, 128, 64, "f32", dict(axes=3, interleaved=True)), (13, 2, 1, 72, 66, "f16", dict(axes=4, interleaved=True, neighbours=True)),
         (30, 2, 1, 128, 128, "f32", dict(far=True)), (30, 2, 1, 128, 128, "f16", dict(far=True, axes=2)), (30, 2, 1, 64, 64, "f32", dict(weight="q")),
         (30, 2, 1, 64, 64, "f32", dict(weight="k", scale=0.75)), (30, 2, 1, 64, 64, "bf16", dict(weight="none", scale=1.5)), (7, 100, 1, 128, 128, "f32", {}),
         (3, 300, 70, 3, 2, "f16", {}), (5000, 2, 1, 64, 64, "f32", {}), (4099, 1, 1, 15, 8, "bf16", {}), (2049, 40, 8, 128, 128, "bf16", {}),
         (1026, 40, 8, 128, 96, "f32", dict(neighbours=True, axes=2)), (4101, 3, 2, 130, 128, "f16", {}), (4097, 1, 0, 200, 24, "f16", dict(norm=False, neighbours=True)),
         (6, 2, 2, 255, 254, "f32", {}), (6, 2, 2, 300, 200, "f16", dict(neighbours=True)), (4100, 4, 4, 40, 8, "f32", dict(neighbours=True)),
         (4200, 4, 4, 24, 8, "bf16", dict(neighbours=True)), (2100, 9, 3, 70, 66, "bf16", {}), (2100, 9, 3, 70, 66, "f32", dict(neighbours=True, axes=2)), (2100, 9, 3, 128, 10, "f16", {}),
         (2100, 5, 1, 512, 2, "f32", {}), (2100, 9, 3, 90, 0, "bf16", {})]


@pytest.mark.parametrize("rows,q_heads,k_heads,D,R,kind,more", CASES)
def test_norm_and_rotation(sess, rows, q_heads, k_heads, D, R, kind, more):
    case = Case(rows, q_heads, k_heads, D, R, kind, **more)
    outs = [None if x is None else torch.full_like(x, 77.0) for x in (case.q, case.k)]
    case.call(sess, case.q, case.k, *outs)
    done(sess)
    case.check(*outs)
    # in place: the same bits
    here = [None if x is None else x.clone() for x in (case.q, case.k)]
    case.call(sess, *here)
    done(sess)
    assert all(a is None or torch.equal(a, b) for a, b in zip(outs, here))


@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_heads_and_turned_parts_of_every_length(sess, kind, neighbours):
    """Turned and not in any number of values, in place: what no unit holds as a whole is turned and left out once."""
    pairs = [(D, R) for D in range(1, 42) for R in range(0, D + 1, 2)] + [(D, R) for D in (127, 128, 200, 509, 511, 512) for R in (0, 2, 14, 18, 74, 126, 2 * (D // 2) - 2, 2 * (D // 2)) if R <= D]
    for D, R in pairs:
        case = Case(3, 2, 1, D, R, kind, neighbours=neighbours, norm=D % 3 != 0)
        q, k = case.q.clone(), case.k.clone()
        case.call(sess, q, k)
        done(sess)
        case.check(q, k)


@pytest.mark.parametrize("kind,D,R,shift", [("bf16", 128, 128, 0), ("f16", 64, 32, 1), ("f32", 72, 72, 3), ("bf16", 33, 10, 5)])
@pytest.mark.parametrize("rows", [1, 6, 4500])
def test_queries_and_keys_of_a_projection_in_place(sess, kind, D, R, shift, rows):
    """Rows of q, k, v in one buffer, at any alignment: nothing but the queries and keys changes."""
    case = Case(rows, 3, 2, D, R, kind)
    width = 7 * D + 3
    whole = torch.full((rows * width + shift,), 77.0, dtype=TYPES[kind], device="cuda")
    table = whole[shift:].view(rows, width)
    q, k = table[:, :3 * D].unflatten(1, (3, D)), table[:, 3 * D:5 * D].unflatten(1, (2, D))
    q.copy_(case.q)
    k.copy_(case.k)
    case.call(sess, q, k)
    done(sess)
    case.check(q, k)
    assert (whole[:shift] == 77).all() and (table[:, 5 * D:] == 77).all()


@pytest.mark.parametrize("rows", [1, 9, 4500])
def test_heads_that_hold_their_rows(sess, rows):
    """[heads, rows, D] in, with rows behind the last one; both layouts out."""
    case = Case(rows, 3, 2, 64, 64, "bf16", axes=2)
    held = [torch.full((x.shape[1], rows + 5, 64), 77.0, dtype=x.dtype, device="cuda") for x in (case.q, case.k)]
    views = [h[:, :rows].transpose(0, 1) for h in held]
    for v, x in zip(views, (case.q, case.k)):
        v.copy_(x)
    outs = [torch.zeros_like(x) for x in (case.q, case.k)]
    case.call(sess, *views, *outs)
    done(sess)
    case.check(*outs)
    case.call(sess, *views)
    done(sess)
    assert all(torch.equal(v, o) for v, o in zip(views, outs)) and all((h[:, rows:] == 77).all() for h in held)


def test_a_cache_as_the_keys_output(sess):
    """Keys go to their rows of a longer cache, of another pitch; queries stay where they are."""
    rows, at, room = 6, 11, 40
    case = Case(rows, 4, 2, 128, 128, "f16")
    cache = torch.full((2, room, 128), 77.0, dtype=torch.float16, device="cuda")
    q = case.q.clone()
    k_out = cache[:, at:at + rows].transpose(0, 1)
    case.call(sess, q, case.k, None, k_out)
    done(sess)
    case.check(q, k_out)
    assert (cache[:, :at] == 77).all() and (cache[:, at + rows:] == 77).all()


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_infinities_and_nan_stay_in_their_head_or_pair(sess, norm, kind):
    case = Case(4, 3, 2, 64, 32, kind, norm=norm)
    clean = [torch.zeros_like(x) for x in (case.q, case.k)]
    case.call(sess, case.q, case.k, *clean)
    x, y = case.q.clone(), case.k.clone()
    x[1, 2, 5], y[3, 0, 40], x[0, 0, 16] = float("nan"), float("inf"), float("-inf")
    outs = [torch.zeros_like(v) for v in (x, y)]
    case.call(sess, x, y, *outs)
    done(sess)
    q, k = torch.zeros_like(x, dtype=torch.bool), torch.zeros_like(y, dtype=torch.bool)
    if norm:
        q[1, 2] = q[0, 0] = k[3, 0] = True
    else:
        q[1, 2, [5, 21]] = q[0, 0, [0, 16]] = k[3, 0, 40] = True
    assert torch.equal(outs[0][~q], clean[0][~q]) and torch.equal(outs[1][~k], clean[1][~k])
    assert outs[0][1, 2, 5].isnan() and (not norm or outs[0][1, 2].isnan().all()) and (not norm or outs[1][3, 0, 40].isnan()) and (norm or outs[1][3, 0, 40].isinf())


def test_heads_of_zeros_and_of_tiny_values(sess):
    case = Case(3, 2, 1, 128, 128, "f32")
    case.q.zero_()
    case.k.mul_(1e-12)
    case.call(sess, case.q, case.k, *(outs := [torch.full_like(x, 7.0) for x in (case.q, case.k)]))
    done(sess)
    assert (outs[0] == 0).all()
    case.check(*outs)


def test_many_short_rows(sess):
    case = Case(300001, 1, 0, 4, 2, "f16")
    out = torch.zeros_like(case.q)
    case.call(sess, case.q, None, out)
    done(sess)
    case.check(out, None)


def test_rows_further_apart_than_32_bits(sess):
    rows, D, ld = 5, 128, (1 << 29) + 8
    if torch.cuda.mem_get_info()[0] < 1 << 34:
        pytest.skip("no room")
    case = Case(rows, 1, 1, D, D, "bf16")
    whole = torch.empty((rows - 1) * ld + 2 * D, dtype=torch.bfloat16, device="cuda")
    q, k = whole.as_strided((rows, 1, D), (ld, D, 1)), whole.as_strided((rows, 1, D), (ld, D, 1), D)
    q.copy_(case.q)
    k.copy_(case.k)
    case.call(sess, q, k)
    done(sess)
    case.check(q, k)


@pytest.mark.parametrize("rows", [1, 2100])
def test_captured_calls_replay_what_the_eager_call_gives(sess, rows):
    """Another table of axes and other positions in between: the captured call keeps its table and reads its positions anew."""
    case, other = (Case(rows, 8, 2, 128, 128, "bf16", axes=2, interleaved=i, seed=i) for i in (0, 1))
    outs = [torch.zeros_like(x) for x in (case.q, case.k)]
    case.call(sess, case.q, case.k, *outs)
    done(sess)
    assert sess.lib.rk_npu_hip_capture_begin(sess.ctx) == 0
    case_call = dict(norm=True, q_weight=case.wq, k_weight=case.wk, positions=case.positions, inv_freq=case.inv_freq, pair_axis=case.pair_axis)
    ops.heads_norm_rotate(sess, case.q, case.k, *outs, **case_call)
    graph = sess.lib.rk_npu_hip_capture_end(sess.ctx)
    assert graph
    for turn in range(4):
        case.positions.add_(17)
        case.q.copy_(device(case.rng.standard_normal(case.q.shape), "bf16"))
        for o in outs:
            o.fill_(77)
        other.call(sess, other.q.clone(), other.k.clone())
        ready()
        assert sess.lib.rk_npu_hip_graph_launch(sess.ctx, graph) == 0
        done(sess)
        case.check(*outs)
    sess.lib.rk_npu_hip_graph_free(graph)


def test_batches_of_no_rows_write_nothing(sess):
    case = Case(3, 2, 1, 64, 64, "bf16")
    q, k = case.q.clone(), case.k.clone()
    ready()
    ops.heads_norm_rotate(sess, q[:0], k[:0], q_weight=case.wq, positions=case.positions[:, :0], inv_freq=case.inv_freq)
    done(sess)
    assert torch.equal(q, case.q) and torch.equal(k, case.k)


def test_refusals(sess):
    lib, bad = sess.lib, capi.RK_NPU_ERR_PARAM
    rows, D = 4, 16
    case = Case(rows, 2, 1, D, 8, "f16")
    out = [torch.full_like(x, 5.0) for x in (case.q, case.k)]
    ready()

    def call(ctx=sess.ctx, **what):
        a = capi.HeadsArgs()
        lib.rk_npu_heads_args_init(C.byref(a), rows, D)
        base = dict(q_heads=2, k_heads=1, type=1, q_weight=case.wq.data_ptr(), k_weight=case.wk.data_ptr(), q=case.q.data_ptr(), k=case.k.data_ptr(), q_out=out[0].data_ptr(),
                    k_out=out[1].data_ptr(), q_row=2 * D, q_head=D, k_row=D, k_head=D, q_out_row=2 * D, q_out_head=D, k_out_row=D, k_out_head=D, rotary_dim=8,
                    positions=case.positions.data_ptr(), inv_freq=case.inv_freq.data_ptr())
        for name, v in {**base, **what}.items():
            setattr(a, name, v)
        return lib.rk_npu_heads_norm_rotate_device(ctx, C.byref(a))
    table = (C.c_uint8 * 4)(0, 1, 0, 0)
    q, k = case.q.data_ptr(), case.k.data_ptr()
    for wrong in (dict(ctx=None), dict(struct_size=8), dict(rows=-1), dict(rows=2 ** 31 - 1, q_row=D, q_head=2 ** 36, q_out_row=D, q_out_head=2 ** 36, k_heads=0), dict(head_dim=0), dict(head_dim=513, rotary_dim=0, q_row=2000, q_head=600, k_row=600), dict(q_heads=-1), dict(k_heads=-1),
                  dict(q_heads=1 << 21), dict(type=3), dict(type=-1), dict(rotary_dim=7), dict(rotary_dim=-2), dict(rotary_dim=18), dict(axes=0), dict(axes=5), dict(eps=-1.0),
                  dict(eps=float("nan")), dict(norm=0), dict(q=None), dict(k_out=None), dict(q=q + 1), dict(q_head=D - 1), dict(q_row=2 * D - 1), dict(k_row=D - 1),
                  dict(q_out_row=D), dict(q_row=1 << 62), dict(q_row=-32), dict(positions=None), dict(inv_freq=None), dict(positions=case.positions.data_ptr() + 2),
                  dict(inv_freq=case.inv_freq.data_ptr() + 1), dict(position_axis=-1), dict(pair_axis=C.addressof(table)), dict(q_weight=case.wq.data_ptr() + 2),
                  dict(q_out=q + 2), dict(q_out=k), dict(k_out=q), dict(q_out=q, q_out_head=rows * D, q_out_row=D), dict(k_out=out[0].data_ptr() + 2 * D * 7), dict(k_out=case.wq.data_ptr()),
                  dict(q_out=case.positions.data_ptr()), dict(k_out=case.inv_freq.data_ptr())):
        assert call(**wrong) == bad, wrong
    done(sess)
    assert all((x == 5).all() for x in out)
    # nothing to do, and pointers that do not matter
    assert call(rows=0) == 0 and call(q_heads=0, k_heads=0) == 0 and call(rows=0, positions=None, inv_freq=None) == 0
    done(sess)
    assert all((x == 5).all() for x in out)
    assert call(q_heads=0, q=None, q_out=None) == 0 and call(rotary_dim=0, positions=None, inv_freq=None) == 0 and call(pair_axis=C.addressof(table), axes=2, rows=1) == 0
    done(sess)
