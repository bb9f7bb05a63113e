"""Launches go to the current device: tensors of another one are refused, as
their kernels would run beside them, on the current one."""

import pytest
import torch

from voyager_amd import _lib


@pytest.fixture
def two_devices(monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 100 + index, raising=False)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)


def test_another_device_is_refused(two_devices):
    with pytest.raises(RuntimeError, match="cuda:0.*cuda:1"):
        _lib.stream_on(torch.device("cuda", 0))


def test_the_current_one_is_not(two_devices):
    assert _lib.stream_on(torch.device("cuda", 1)) == 101
    assert _lib.stream_on(torch.device("cuda")) == 101


def test_the_host_is(two_devices):
    with pytest.raises(ValueError, match="cuda"):
        _lib.stream_on(torch.device("cpu"))
