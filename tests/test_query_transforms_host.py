"""CPU tests of what the query operators refuse of torch's transforms, before anything else is looked at."""
import pytest
import torch
from torch.autograd import forward_ad

from flashbev_b200 import add_rms_norm, cross_attention, flash_bevpool, rotary_axes

CALLS = [lambda x: cross_attention(x, x, x), lambda x: rotary_axes(x, torch.zeros(2, 1), (4,)), lambda x: add_rms_norm(x)[0],
         lambda x: add_rms_norm(x, quantize=True)[1]]


@pytest.mark.parametrize("call", CALLS, ids=["attention", "rotary", "norm", "norm_8bit"])
@pytest.mark.parametrize("grad", [False, True])
def test_tracing_is_refused(call, grad):
    x = torch.zeros(1, 2, 2, 8, requires_grad=grad)
    with pytest.raises(RuntimeError, match="trace"):
        torch.jit.trace(call, x, check_trace=False)


@pytest.mark.parametrize("call", CALLS, ids=["attention", "rotary", "norm", "norm_8bit"])
def test_forward_mode_is_refused(call):
    x = torch.zeros(1, 2, 2, 8)
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(forward_ad.make_dual(x, torch.ones_like(x)))
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            call(forward_ad.make_dual(x, torch.ones_like(x)))
        with pytest.raises(RuntimeError, match="CUDA"):  # no tangent: the next check
            call(x)


@pytest.mark.parametrize("which", ["image_feats", "depth_params"])
def test_pooling_refuses_forward_mode(which):
    inp = {"image_feats": torch.zeros(1, 1, 2, 2, 8), "depth_params": torch.ones(1, 1, 2, 2, 2),
           "projection_matrices": torch.zeros(1, 1, 3, 4), "feature_size": torch.full((1, 1, 2), 2, dtype=torch.int32),
           "image_size": torch.tensor([4, 4], dtype=torch.int32), "roi_range": torch.zeros(6),
           "grid_size": torch.tensor([2, 2, 2], dtype=torch.int32)}
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="CUDA"):
            flash_bevpool(**inp)
        inp[which] = forward_ad.make_dual(inp[which], torch.ones_like(inp[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            flash_bevpool(**inp)


def test_which_strides_are_read_in_place():
    from flashbev_b200.query_ops import _operand, _taken
    x = torch.arange(2 * 3 * 2 * 16 + 64, dtype=torch.bfloat16)
    whole, odd = x.as_strided((2, 3, 2, 16), (96, 32, 16, 1)), x.as_strided((2, 3, 2, 16), (100, 32, 16, 1))
    assert _taken(whole) and _taken(whole, shared_batch=True)
    one = x.as_strided((1, 3, 2, 16), (100, 32, 16, 1))  # the stride of a dimension of one is not used
    assert _taken(one) and _taken(one.expand(2, -1, -1, -1), shared_batch=True) and not _taken(one.expand(2, -1, -1, -1))
    for shared in (False, True):  # samples that are not whole 16 bytes apart: a copy, not the kernels of odd widths
        assert not _taken(odd, shared_batch=shared)
        got = _operand(odd, shared_batch=shared)
        assert got is not odd and got.is_contiguous() and torch.equal(got, odd)
    assert _taken(odd.float())
