"""What the Python wrappers of the MX4 calls decide before anything reaches the device."""
import pytest
import torch

from rknpu2_matmul_open_amd import ops


class OnDevice:
    """What the wrappers look at in a tensor on the device."""

    def __init__(self, t, index=None):
        self.dtype, self.shape, self.is_cuda, self.stride, self.data_ptr, self.is_contiguous, self.reshape = t.dtype, t.shape, True, t.stride, t.data_ptr, t.is_contiguous, t.reshape
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
