"""What the Python wrappers of the G4 and heads calls decide before anything reaches the device."""
import numpy as np
import pytest
import torch

from rknpu2_matmul_open_amd import capi, ops
from tests.test_mx4_wrappers import Session


class OnDevice:
    """What the wrappers look at in a tensor on the device."""

    def __init__(self, t, index=1):
        self.dtype, self.shape, self.is_cuda, self.stride, self.data_ptr, self.is_contiguous = t.dtype, t.shape, True, t.stride, t.data_ptr, t.is_contiguous
        self.device = torch.device("cuda", index)


def tensor(*shape, dtype=torch.uint8, index=1):
    return OnDevice(torch.zeros(*shape, dtype=dtype), index)


def test_weights_are_checked():
    K, N, group = 75, 4, 32
    s = Session()
    half = tensor(N, 3, dtype=torch.float16)
    ops.G4Weights.from_device(s, K, N, group, tensor(N, 38), half)
    ops.G4Weights.from_device(s, K, N, group, tensor(N, 38), tensor(N, 3, dtype=torch.bfloat16), tensor(N, 3))
    assert s.lib.calls == ["rk_npu_g4_weights_create_device"] * 2
    ops.G4Weights(s, K, N, group, np.zeros((N, 38), np.uint8), np.zeros((N, 3), np.float16))
    ops.G4Weights(s, K, N, group, np.zeros((N, 38), np.uint8), np.zeros((N, 3), np.uint16), np.zeros((N, 3), np.uint8), scale_type=capi.MX4_BF16)
    assert s.lib.calls[2:] == ["rk_npu_g4_weights_create"] * 2
    strided = OnDevice(torch.zeros(N, 76, dtype=torch.uint8)[:, ::2])
    for args in ((tensor(N, 37), half), (tensor(N - 1, 38), half), (tensor(N, 38), tensor(N, 2, dtype=torch.float16)), (tensor(N, 38, dtype=torch.int8), half), (strided, half),
                 (tensor(N, 38, index=0), half), (tensor(N, 38), tensor(N, 3, dtype=torch.float16, index=0)), (tensor(N, 38), half, tensor(N, 2)),
                 (tensor(N, 38), half, tensor(N, 3, index=0)), (tensor(N, 38), half, tensor(N, 3, dtype=torch.int32)), (torch.zeros(N, 38, dtype=torch.uint8), half)):
        with pytest.raises(ValueError):
            ops.G4Weights.from_device(s, K, N, group, *args)
    with pytest.raises(TypeError):
        ops.G4Weights.from_device(s, K, N, group, tensor(N, 38), tensor(N, 3, dtype=torch.float32))
    for codes, scales in ((np.zeros((N, 76), np.uint8)[:, ::2], np.zeros((N, 3), np.float16)), (np.zeros((N, 38), np.uint8), np.zeros((N, 4), np.float16))):
        with pytest.raises(ValueError):
            ops.G4Weights(s, K, N, group, codes, scales)
    with pytest.raises(ValueError):
        ops.G4Weights(s, K, N, group, torch.zeros((N, 38), dtype=torch.uint8), np.zeros((N, 3), np.float16))
    with pytest.raises(ValueError):
        ops.G4Weights(s, K, N, 0, np.zeros((N, 38), np.uint8), np.zeros((N, 3), np.float16))
    assert len(s.lib.calls) == 4


def test_runs_are_checked():
    s = Session()
    ws = ops.G4Workspace(s, 8, 40, 64)

    class W:
        N, h = 64, None
    x = lambda *shape, dtype=torch.float16, index=1: tensor(*shape, dtype=dtype, index=index)  # noqa: E731
    ws.run(W, x(3, 40), x(3, 64, dtype=torch.float32))
    ws.run_swiglu(W, x(3, 40, dtype=torch.bfloat16), x(3, 32))
    assert s.lib.calls[1:] == ["rk_npu_g4_run_device", "rk_npu_g4_run_swiglu_device"]
    for a, c in ((x(3, 41), x(3, 64)), (x(3, 40), x(3, 63)), (x(3, 40), x(4, 64)), (x(3, 40, index=0), x(3, 64)), (x(3, 40), x(3, 64, index=0))):
        with pytest.raises(ValueError):
            ws.run(W, a, c)
    with pytest.raises(ValueError):
        ws.run_swiglu(W, x(3, 40), x(3, 64))
    for a, c in ((x(3, 40, dtype=torch.float32), x(3, 64)), (x(3, 40, dtype=torch.float64), x(3, 64)), (x(3, 40), x(3, 64, dtype=torch.int32))):
        with pytest.raises(TypeError):
            ws.run(W, a, c)
    assert len(s.lib.calls) == 3


def test_pair_axes():
    assert ops.pair_axes([2, 3, 1]) == [0, 0, 1, 1, 1, 2]
    assert ops.pair_axes([2, 3, 1], interleaved=True) == [0, 1, 2, 0, 1, 1]
    assert ops.pair_axes([0, 2]) == [1, 1] and ops.pair_axes([]) == []


def test_heads_are_checked():
    s = Session()
    rows, D = 5, 16
    t = lambda heads, dtype=torch.float16, index=1, rows=rows, D=D: tensor(rows, heads, D, dtype=dtype, index=index)  # noqa: E731
    channel = lambda n, index=1, dtype=torch.float32: tensor(n, dtype=dtype, index=index)  # noqa: E731
    pos = lambda *shape, dtype=torch.int32, index=1: tensor(*shape, dtype=dtype, index=index)  # noqa: E731
    ops.heads_norm_rotate(s, t(4), t(2))
    ops.heads_norm_rotate(s, t(4), None, q_weight=channel(D))
    ops.heads_norm_rotate(s, None, t(2), k_out=t(2), norm=False, positions=pos(rows), inv_freq=channel(8))
    ops.heads_norm_rotate(s, t(4), t(2), positions=pos(3, rows), inv_freq=channel(8), pair_axis=[0, 0, 1, 1, 2, 2, 2, 0])
    calls = [c for c in s.lib.calls if c == "rk_npu_heads_norm_rotate_device"]
    assert len(calls) == 4
    a = ops.heads_args(s, t(4), t(2), positions=pos(3, rows), inv_freq=channel(6), pair_axis=[2] * 6)
    assert (a.q_heads, a.k_heads, a.rotary_dim, a.axes, a.q_row, a.q_head, a.q, a.type) == (4, 2, 12, 3, 64, 16, a.q_out, capi.MX4_F16)
    for what in (lambda: ops.heads_norm_rotate(s, None, None), lambda: ops.heads_norm_rotate(s, t(4), t(2, D=18)), lambda: ops.heads_norm_rotate(s, t(4), t(2, rows=4)),
                 lambda: ops.heads_norm_rotate(s, t(4), t(2, dtype=torch.bfloat16)), lambda: ops.heads_norm_rotate(s, t(4), t(2), q_out=t(3)),
                 lambda: ops.heads_norm_rotate(s, t(4), None, k_out=t(2)), lambda: ops.heads_norm_rotate(s, t(4, index=0), t(2)),
                 lambda: ops.heads_norm_rotate(s, t(4), t(2), k_out=t(2, index=0)), lambda: ops.heads_norm_rotate(s, t(4), t(2), q_weight=channel(15)),
                 lambda: ops.heads_norm_rotate(s, t(4), t(2), k_weight=channel(D, index=0)), lambda: ops.heads_norm_rotate(s, t(4), t(2), positions=pos(rows)),
                 lambda: ops.heads_norm_rotate(s, t(4), t(2), inv_freq=channel(8)), lambda: ops.heads_norm_rotate(s, t(4), t(2), pair_axis=[0] * 8),
                 lambda: ops.heads_norm_rotate(s, t(4), t(2), positions=pos(rows - 1), inv_freq=channel(8)),
                 lambda: ops.heads_norm_rotate(s, t(4), t(2), positions=pos(rows, dtype=torch.int64), inv_freq=channel(8)),
                 lambda: ops.heads_norm_rotate(s, t(4), t(2), positions=pos(rows, index=0), inv_freq=channel(8)),
                 lambda: ops.heads_norm_rotate(s, t(4), t(2), positions=pos(2, rows), inv_freq=channel(8), pair_axis=[0] * 7),
                 lambda: ops.heads_norm_rotate(s, t(4), t(2), positions=pos(2, rows), inv_freq=channel(8), pair_axis=[2] * 8),
                 lambda: ops.heads_norm_rotate(s, OnDevice(torch.zeros(rows, 4, 2 * D, dtype=torch.float16)[:, :, ::2]), None)):
        with pytest.raises(ValueError):
            what()
    with pytest.raises(TypeError):
        ops.heads_norm_rotate(s, t(4, dtype=torch.float64), None)
    assert [c for c in s.lib.calls if c == "rk_npu_heads_norm_rotate_device"] == calls
