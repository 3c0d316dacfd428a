"""GPU tests of the device's status word: a first call that a graph captures neither owns nor clears it, and what device_status
reads of it."""
import os
import subprocess
import sys

import pytest
import torch

from flashbev_b200 import DeviceStatus, device_status
from flashbev_b200.flash_bevpool import status_word

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# a process of its own: the operators' first call on the device is a captured one
CAPTURED_FIRST = """
import torch
from flashbev_b200 import cross_attention
from flashbev_b200.flash_bevpool import status_word
dev = torch.device("cuda", 0)
q = torch.randn(1, 3, 2, 64, device=dev).bfloat16()
k = torch.randn(1, 700, 2, 64, device=dev).bfloat16()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = cross_attention(q, k, k)
plain = cross_attention(q, k, k)   # the same plan, outside
word = status_word(dev)
assert int(word.item()) == 0       # before any replay
word |= 2                          # raised by another call
for _ in range(2):
    graph.replay()
torch.cuda.synchronize()
assert int(word.item()) == 2, "a replay cleared the word"
assert torch.equal(out, plain)
with torch.inference_mode():
    assert status_word(dev) is word
print("fine")
"""


def test_first_call_on_the_device_is_captured(cuda_device):
    r = subprocess.run([sys.executable, "-c", CAPTURED_FIRST], cwd=ROOT, capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and r.stdout.strip() == "fine", r.stderr[-2000:]


def test_device_status(cuda_device):
    word = status_word(cuda_device)
    before = device_status(cuda_device, clear=True)
    assert before == DeviceStatus.OK and device_status() == DeviceStatus.OK
    word |= 3
    assert device_status() == DeviceStatus.BAD_FEATURE_SIZE | DeviceStatus.TIMEOUT
    assert device_status(0, clear=True) & DeviceStatus.TIMEOUT and device_status("cuda:0") == 0
    with torch.inference_mode():
        word |= 2
        assert device_status(clear=True) == DeviceStatus.TIMEOUT and not device_status(clear=True)
    graph = torch.cuda.CUDAGraph()
    x = torch.zeros(1, device=cuda_device)
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="capture"):
            device_status()
        x += 1
    graph.replay()
    torch.cuda.synchronize()
    assert float(x) == 1.0
