"""GPU tests of modules that are evaluated under torch.inference_mode() before they are trained."""
import pytest
import torch

from tests.test_gpu_camera_attention import _block

pytestmark = pytest.mark.gpu


def test_block_is_trained_after_inference(cuda_device):
    m, bev, features = _block(cuda_device)
    with torch.inference_mode():
        before = m(bev, features, 6)
    out = m(bev, features, 6)
    out.square().sum().backward()
    assert torch.equal(out.detach(), before)
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in m.parameters())
