"""What the Python wrappers of the MX4 calls decide before anything reaches the device."""
import pytest
import torch

from rknpu2_matmul_open_amd import ops


class OnDevice:
    """What the wrappers look at in a tensor on the device."""

    def __init__(self, t, index=None):
        self.dtype, self.shape, self.is_cuda, self.stride, self.data_ptr, self.is_contiguous = t.dtype, t.shape, True, t.stride, t.data_ptr, t.is_contiguous
        self.reshape = lambda *shape: OnDevice(t.reshape(*shape), index)
        if index is not None:
            self.device = torch.device("cuda", index)


class Weights:
    N, gate_up, h = 64, False, None


def workspace(staged):
    ws = ops.MX4Workspace.__new__(ops.MX4Workspace)
    ws.K, ws.staged, ws.lib, ws.h = 40, staged, None, None # (nothing may be called)
    return ws


def test_an_empty_batch_was_staged():
    """No rows staged is a batch without results; nothing staged is an error."""
    workspace(0).run_staged(Weights, OnDevice(torch.zeros(0, 64)))
    for staged, rows in ((None, 0), (None, 3), (0, 3), (5, 0)):
        with pytest.raises(ValueError):
            workspace(staged).run_staged(Weights, OnDevice(torch.zeros(rows, 64)))
    with pytest.raises(ValueError): # (an empty result of other columns)
        workspace(0).run_staged(Weights, OnDevice(torch.zeros(0, 63)))


class Lib:
    """Calls are noted, not made."""

    def __init__(self):
        self.calls = []

    def rk_npu_hip_device(self, ctx):
        return 1

    def __getattr__(self, name):
        def call(*args):
            self.calls.append(name)
            return 4096 if "create" in name else 0
        return call


class Session:
    def __init__(self):
        self.lib, self.ctx, self.domain = Lib(), None, None


def test_weights_from_device_tensors_are_checked():
    """Tensors that quantization fills are taken, and addresses as they are; short, strided, host and other devices' tensors are refused."""
    K, N = 40, 4
    new = lambda rows, width, index=1, dtype=torch.uint8: OnDevice(torch.zeros(rows, width, dtype=dtype), index)  # noqa: E731
    s = Session()
    ops.MX4Weights.from_device(s, K, N, new(N, 32), new(N, 2))
    ops.MX4Weights.from_device(s, K, N, new(N, 32), 4096)
    ops.MX4Weights.from_device(s, K, N, 4096, 8192)
    assert s.lib.calls == ["rk_npu_mx4_weights_create_device"] * 3
    strided = OnDevice(torch.zeros(N, 64, dtype=torch.uint8)[:, ::2], 1)
    for codes, scales in ((new(N, 16), new(N, 2)), (new(N - 1, 32), new(N, 2)), (new(N, 32), new(N, 1)), (new(N, 32, dtype=torch.int8), new(N, 2)), (strided, new(N, 2)),
                          (new(N, 32, index=0), new(N, 2)), (new(N, 32), new(N, 2, index=0)), (torch.zeros(N, 32, dtype=torch.uint8), new(N, 2))):
        with pytest.raises(ValueError):
            ops.MX4Weights.from_device(s, K, N, codes, scales)
    assert len(s.lib.calls) == 3


def test_tensors_of_another_device_are_refused():
    """The context is on device 1: every wrapper takes tensors there and none of device 0, wherever they stand."""
    s = Session()
    rows, D = 3, 64
    t = lambda width=D, index=1, dtype=torch.float32: OnDevice(torch.zeros(rows, width, dtype=dtype), index)  # noqa: E731
    channel = lambda index: OnDevice(torch.zeros(D), index)  # noqa: E731
    byte = lambda width, index: t(width, index, torch.uint8)  # noqa: E731
    ws, other = ops.MX4Workspace(s, 8, D, D), ops.MX4Workspace(s, 8, D, D)

    class W:
        N, gate_up, h = D, False, None

    class Pair:
        N, gate_up, h = 2 * D, True, None
    calls = {
        "mx4_quantize": lambda i: ops.mx4_quantize(s, t(index=i[0]), byte(32, i[1]), byte(2, i[2])),
        "mx4_dequantize": lambda i: ops.mx4_dequantize(s, byte(32, i[0]), byte(2, i[1]), t(index=i[2])),
        "run": lambda i: ws.run(W, t(index=i[0]), t(index=i[1])),
        "run_swiglu": lambda i: ws.run_swiglu(Pair, t(index=i[0]), t(index=i[1])),
        "stage": lambda i: ws.stage(t(index=i[0])),
        "run_staged": lambda i: (ws.stage(t()), ws.run_staged(W, t(index=i[0]))),
        "mx4_ffn": lambda i: ops.mx4_ffn(ws, Pair, other, W, t(index=i[0]), t(index=i[1])),
        "block_norm": lambda i: ops.block_norm(s, t(index=i[0]), t(index=i[1]), after=channel(i[2]), gate=channel(i[3]), weight=channel(i[4]), stream_out=t(index=i[5]),
                                               y=t(index=i[6])),
        "block_norm, rows of the gate": lambda i: ops.block_norm(s, t(), t(), gate=t(index=i[0]), y=t()),
        "mx4_ffn_block": lambda i: ops.mx4_ffn_block(ws, Pair, other, W, t(index=i[0]), t(index=i[1]), weight=channel(i[2]), after=channel(i[3]), gate=channel(i[4]),
                                                     stream_out=t(index=i[5]), y=t(index=i[6]), next_weight=channel(i[7])),
    }
    places = {"mx4_quantize": 3, "mx4_dequantize": 3, "run": 2, "run_swiglu": 2, "stage": 1, "run_staged": 1, "mx4_ffn": 2, "block_norm": 7, "block_norm, rows of the gate": 1,
              "mx4_ffn_block": 8}
    for name, call in calls.items():
        call([1] * places[name])
        for wrong in range(places[name]):
            with pytest.raises(ValueError):
                call([0 if k == wrong else 1 for k in range(places[name])])
