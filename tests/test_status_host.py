"""CPU test of device_status's refusals and flags."""
import pytest
import torch

from flashbev_b200 import DeviceStatus, _lib, device_status


def test_flags_are_the_headers():
    assert int(DeviceStatus.BAD_FEATURE_SIZE) == _lib.DEV_BAD_FEATURE_SIZE and int(DeviceStatus.TIMEOUT) == _lib.DEV_TIMEOUT
    assert not DeviceStatus.OK


def test_device_status_wants_a_cuda_device():
    for device in ("cpu", torch.device("cpu"), "meta"):
        with pytest.raises(ValueError, match="CUDA"):
            device_status(device)
