"""GPU tests of CameraAttention and SamplingVT(attention_heads=n) under torch.autocast: float32 parameters, products in 16 bits."""
import pytest
import torch

from flashbev_b200 import SamplingVT, synth
from tests.test_gpu_camera_attention import GRID, _block, _double, _far, _plain

pytestmark = pytest.mark.gpu

# as for the block in 16 bits: tensors are rounded between its ten stages (bfloat16 2^-8, float16 2^-11 each, independent),
# the parameters besides; the largest value of a tensor is the measure
TOL = {torch.bfloat16: 2.0 ** -4, torch.float16: 2.0 ** -7}
TYPES = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])


@TYPES
@pytest.mark.parametrize("features_in", ["float32", "16 bits"])
@pytest.mark.parametrize("masked", [False, True])
def test_block_under_autocast(cuda_device, dtype, features_in, masked):
    m, bev, features = _block(cuda_device)
    kind = torch.float32 if features_in == "float32" else dtype
    bev, features = bev.to(kind).requires_grad_(), features.to(kind).requires_grad_()
    mask = None
    if masked:
        mask = torch.ones(2, 6, dtype=torch.bool, device=cuda_device)
        mask[0, 2] = mask[1, 5] = False
    with torch.autocast("cuda", dtype=dtype):
        out = m(bev, features, 6, mask)
    assert out.dtype == kind and out.shape == bev.shape
    up = torch.randn(out.shape, generator=torch.Generator(device="cuda").manual_seed(1), device=cuda_device).to(kind)
    names = [n for n, _ in m.named_parameters()]
    grads = torch.autograd.grad(out, [bev, features, *m.parameters()], up)
    assert all(g.dtype == t.dtype for g, t in zip(grads, [bev, features, *m.parameters()]))
    d, bd, fd = _double(m, bev, features)
    ref = _plain(d, bd, fd, 6, mask)
    want = torch.autograd.grad(ref, [bd, fd, *(d[n] for n in names)], up.double())
    assert _far(out, ref) <= TOL[dtype]
    for n, a, b in zip(["bev", "features", *names], grads, want):
        assert _far(a, b) <= TOL[dtype], n


@TYPES
def test_sampling_vt_under_autocast(cuda_device, dtype):
    inputs, image = synth.module_inputs(B=2, N=6, C=32, H=8, W=22, seed=5)
    inputs = [t.to(cuda_device) for t in inputs]
    torch.manual_seed(0)
    plain = SamplingVT(GRID, image, in_channels=32, out_channels=16).to(cuda_device)
    m = SamplingVT(GRID, image, in_channels=32, out_channels=16, attention_heads=2).to(cuda_device)
    m.load_state_dict(plain.state_dict(), strict=False)
    with torch.autocast("cuda", dtype=dtype), torch.no_grad():
        a, b = plain(inputs)[0], m(inputs)[0]
    assert a.dtype == b.dtype == dtype and torch.equal(a, b)  # the block starts as the identity
    with torch.no_grad():
        m.camera_attention.to_out.weight.normal_(std=0.2)
    with torch.autocast("cuda", dtype=dtype):
        out, _ = m(inputs)
    assert out.dtype == dtype and out.shape == a.shape and not torch.equal(out, a)
    out.float().square().mean().backward()
    assert all(p.grad is not None and p.grad.dtype == torch.float32 and torch.isfinite(p.grad).all() for p in m.parameters())
