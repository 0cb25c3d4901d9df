"""CPU: the device-side step state of muon_step_ and adam_step_multi_ is checked before its pointer goes to a kernel."""
import ctypes
import importlib

import pytest
import torch


@pytest.fixture(scope="module")
def S():
    import spin_nerf_amd as S
    return S


class OnDevice:
    """a tensor on a device for what the check asks of it"""

    def __init__(self, t, index):
        self.t, self.index = t, index
        self.is_cuda = index >= 0

    def get_device(self):
        return self.index

    def __getattr__(self, name):
        return getattr(self.t, name)


def test_a_state_that_a_kernel_cannot_read_is_refused(S):
    ops = importlib.import_module("spin-nerf_amd.ops")
    n = ctypes.sizeof(S._lib.StepState)
    good = torch.zeros(n, dtype=torch.uint8)
    assert ops.state_ptr("f", None, 0) is None
    assert ops.state_ptr("f", OnDevice(good, 0), 0).value == good.data_ptr()
    assert ops.state_ptr("f", OnDevice(torch.zeros(n // 8, dtype=torch.int64), 1), 1) is not None
    with pytest.raises(S.HipLibraryError, match="CPU tensor"):
        ops.state_ptr("f", good, 0)
    with pytest.raises(ValueError, match="cuda:0"):
        ops.state_ptr("f", OnDevice(good, 1), 0)
    for short in (good[:-1], good[:0], torch.zeros(1), torch.zeros(2 * n, dtype=torch.uint8)[::2], torch.zeros(n + 4, dtype=torch.uint8)[4:]):
        with pytest.raises(ValueError, match="snr_step_state"):
            ops.state_ptr("f", OnDevice(short, 0), 0)
