"""check_kernels against a fake of the library's flags: no kernel is made to give up."""
import ctypes

import pytest
import torch

from llima_b200 import _native as N
from llima_b200 import fp8


class FakeLib:
    def __init__(self, flags, status=0):
        self.flags, self.status, self.calls = dict(flags), status, []

    def gq_kernel_errors(self, device, clear, out):
        self.calls.append((device, clear))
        ctypes.cast(out, ctypes.POINTER(ctypes.c_uint32))[0] = self.flags.get(device, 0)
        if clear:
            self.flags[device] = 0
        return self.status

    def gq_strerror(self, status):
        return b"fake"

    def gq_last_cuda_error(self):
        return 700


@pytest.fixture
def fake(monkeypatch):
    waited = []
    monkeypatch.setattr(torch.cuda, "synchronize", waited.append)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 2)

    def use(*args, **kwargs):
        lib = FakeLib(*args, **kwargs)
        monkeypatch.setattr(N, "lib", lambda: lib)
        monkeypatch.setattr(N, "_lib", lib)
        return lib, waited

    return use


@pytest.mark.parametrize("device,index", [(None, 2), (1, 1), ("cuda:3", 3), ("cuda", 2), (torch.device("cuda", 0), 0), (torch.device("cuda"), 2)])
def test_flags_of_the_device_are_read_cleared_and_raised(fake, device, index):
    lib, waited = fake({index: 1})
    with pytest.raises(RuntimeError, match=f"cuda:{index} gave up"):
        fp8.check_kernels(device)
    fp8.check_kernels(device)
    assert lib.calls == [(index, 1)] * 2 and waited == [device] * 2     # after the device's work


def test_other_devices_flags_are_left(fake):
    lib, _ = fake({0: 1})
    fp8.check_kernels(1)
    assert lib.flags[0] == 1


def test_a_failed_reading_is_an_error(fake):
    fake({}, status=-6)
    with pytest.raises(N.GqError):
        fp8.check_kernels(0)
