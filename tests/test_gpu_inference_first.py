"""GPU tests of modules that are evaluated under torch.inference_mode() before they are trained."""
import pytest
import torch

from flashbev_b200 import SamplingVT, synth
from tests.test_gpu_camera_attention import GRID, _block

pytestmark = pytest.mark.gpu


def test_block_is_trained_after_inference(cuda_device):
    m, bev, features = _block(cuda_device)
    with torch.inference_mode():
        before = m(bev, features, 6)
    out = m(bev, features, 6)
    out.square().sum().backward()
    assert torch.equal(out.detach(), before)
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in m.parameters())


@pytest.mark.parametrize("heads", [0, 2])
def test_sampling_vt_is_trained_after_inference(cuda_device, heads):
    inputs, image = synth.module_inputs(B=2, N=6, C=32, H=8, W=22, seed=5)
    inputs = [t.to(cuda_device) for t in inputs]
    m = SamplingVT(GRID, image, in_channels=32, out_channels=16, attention_heads=heads).to(cuda_device)
    with torch.inference_mode():
        before = m(inputs)[0]
    out, _ = m(inputs)
    out.square().sum().backward()
    assert torch.equal(out.detach(), before)
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in m.parameters())
