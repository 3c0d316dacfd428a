"""GPU tests of refusals that must not depend on the calls before."""
import pytest
import torch

from flashbev_b200 import rotary_axes

pytestmark = pytest.mark.gpu


def test_sections_that_equal_accepted_ones(cuda_device):
    x, p = torch.randn(2, 5, 3, 32, device=cuda_device), torch.randn(5, 2, device=cuda_device)
    for bad in ((8.0, 8), (8, 8.0), (torch.tensor(8), 8)):
        with pytest.raises(ValueError, match="whole"):
            rotary_axes(x, p, bad)
    want = rotary_axes(x, p, (8, 8))
    for bad in ((8.0, 8), (8, 8.0), (torch.tensor(8), 8)):
        with pytest.raises(ValueError, match="whole"):
            rotary_axes(x, p, bad)
    assert torch.equal(rotary_axes(x, p, [8, 8], base=10000, interleaved=0), want)
