"""GPU tests of the query operators together, as SamplingVT(attention_heads=n) runs them: against the same block written in
plain float64 operations, with all gradients, with a missing camera, in 16 bits and captured in a graph."""
import math

import pytest
import torch

from flashbev_b200 import CameraAttention, SamplingVT, synth

pytestmark = pytest.mark.gpu

GRID = {"x": [-20.0, 20.0, 1.0], "y": [-16.0, 16.0, 1.0], "z": [-4.0, 2.0, 1.0], "depth": [1.0, 60.0, 1.0]}


def _norm(x, w):
    return x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w


def _rotary(x, pos, sections):
    axis = [a for a, s in enumerate(sections) for _ in range(s)]
    freq = torch.tensor([10000.0 ** (-j / s) for s in sections for j in range(s)], dtype=torch.float64, device=x.device)
    ang = (pos.double()[:, axis] * freq).view(1, -1, 1, len(axis))
    a, b = x.chunk(2, dim=-1)
    return torch.cat([a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()], dim=-1)


def _plain(m, bev, features, cameras, camera_mask=None):
    """The block in float64 from elementary operations, differentiable."""
    B, C, Y, X = bev.shape
    h, w = features.shape[-2:]
    x = bev.permute(0, 2, 3, 1).reshape(B, Y * X, C)
    t = features.permute(0, 2, 3, 1).reshape(B, cameras * h * w, -1)
    q = (_norm(x, m["norm_attention"]) @ m["to_q.weight"].T).view(B, Y * X, -1, m["width"])
    kv = (t @ m["to_kv.weight"].T).view(B, cameras * h * w, 2, -1, m["width"])
    pairs = m["width"] // 2
    q = _rotary(q, m["cells"], (pairs - pairs // 2, pairs // 2))
    k = _rotary(kv[:, :, 0], m["tokens"], (pairs - 2 * (pairs // 3), pairs // 3, pairs // 3))
    group = q.shape[2] // k.shape[2]
    k, v = k.repeat_interleave(group, 2), kv[:, :, 1].repeat_interleave(group, 2)
    s = torch.einsum("blhd,bjhd->bhlj", q, k) / math.sqrt(m["width"])
    if camera_mask is not None:
        s = s.masked_fill(~camera_mask.repeat_interleave(h * w, 1).view(B, 1, 1, -1), -math.inf)
    a = torch.einsum("bhlj,bjhd->blhd", torch.softmax(s, -1), v).reshape(B, Y * X, C)
    x = x + a @ m["to_out.weight"].T
    y = _norm(x, m["norm_forward"])
    x = x + torch.nn.functional.gelu(y @ m["widen.weight"].T + m["widen.bias"]) @ m["narrow.weight"].T + m["narrow.bias"]
    return x.view(B, Y, X, C).permute(0, 3, 1, 2)


def _block(device, channels=32, heads=4, key_heads=2, seed=3):
    g = torch.Generator().manual_seed(seed)
    cells = torch.stack(torch.meshgrid(torch.arange(20) - 9.5, torch.arange(24) - 11.5, indexing="ij"), -1).view(-1, 2)
    m = CameraAttention(channels, channels, heads, cells, key_heads=key_heads)
    with torch.no_grad():
        for n, p in m.named_parameters():
            base = 1.0 if n.startswith("norm") else 0.0
            p.copy_(base + torch.randn(p.shape, generator=g) * (0.1 if base else 1 / math.sqrt(p.shape[-1])))
    bev = torch.randn(2, channels, 20, 24, generator=g)
    features = torch.randn(2 * 6, channels, 4, 11, generator=g)
    return m.to(device), bev.to(device), features.to(device)


def _double(m, bev, features):
    d = {n: p.detach().double().requires_grad_() for n, p in m.named_parameters()}
    cells, tokens = m._positions(bev.device, 6, *features.shape[-2:])
    d |= {"width": m.width, "cells": cells, "tokens": tokens}
    return d, bev.detach().double().requires_grad_(), features.detach().double().requires_grad_()


# Errors are compared with the largest value of a tensor.  float32: each of the block's ten stages rounds sums of up to some
# hundred products (2^-24 each, 2^-18 of the largest term for the sum) and its gain is of the order of one: 2^-14 leaves a
# factor of two.  bfloat16: tensors are rounded between the stages (2^-8 each, independent): 2^-4 in the same way.
TOL = {torch.float32: 2.0 ** -14, torch.bfloat16: 2.0 ** -4}


def _far(a, b):
    a, b = a.detach(), b.detach()
    return float((a.double() - b).abs().max() / b.abs().max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("masked", [False, True])
def test_block_against_its_plain_form(cuda_device, dtype, masked):
    m, bev, features = _block(cuda_device)
    m = m.to(dtype)
    bev, features = bev.to(dtype).requires_grad_(), features.to(dtype).requires_grad_()
    mask = None
    if masked:
        mask = torch.ones(2, 6, dtype=torch.bool, device=cuda_device)
        mask[0, 2] = mask[1, 5] = False
    out = m(bev, features, 6, mask)
    assert out.shape == bev.shape and out.dtype == dtype
    up = torch.randn(out.shape, generator=torch.Generator(device="cuda").manual_seed(1), device=cuda_device).to(dtype)
    names = [n for n, _ in m.named_parameters()]
    grads = torch.autograd.grad(out, [bev, features, *m.parameters()], up)
    d, bd, fd = _double(m, bev, features)
    ref = _plain(d, bd, fd, 6, mask)
    want = torch.autograd.grad(ref, [bd, fd, *(d[n] for n in names)], up.double())
    assert _far(out, ref) <= TOL[dtype]
    for n, a, b in zip(["bev", "features", *names], grads, want):
        assert _far(a, b) <= TOL[dtype], n


def test_block_captured_in_a_graph(cuda_device):
    m, bev, features = _block(cuda_device)
    bev.requires_grad_()
    up = torch.ones_like(bev)

    def step():
        out = m(bev, features, 6)
        return [t.detach() for t in (out, *torch.autograd.grad(out, [bev, *m.parameters()], up))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for t in got:
        t.zero_()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    # the operators are the same from run to run; the library's matrix products may take another algorithm under capture
    for a, b in zip(got, want):
        assert _far(a, b.double()) <= TOL[torch.float32]


def test_sampling_vt_with_attention(cuda_device):
    inputs, image = synth.module_inputs(B=2, N=6, C=32, H=8, W=22, seed=5)
    inputs = [t.to(cuda_device) for t in inputs]
    torch.manual_seed(0)
    plain = SamplingVT(GRID, image, in_channels=32, out_channels=16).to(cuda_device)
    m = SamplingVT(GRID, image, in_channels=32, out_channels=16, attention_heads=2).to(cuda_device)
    missing, unexpected = m.load_state_dict(plain.state_dict(), strict=False)
    assert not unexpected and all(k.startswith("camera_attention.") for k in missing)
    with torch.no_grad():
        a, b = plain(inputs)[0], m(inputs)[0]
    assert torch.equal(a, b)  # the block starts as the identity
    with torch.no_grad():
        m.camera_attention.to_out.weight.normal_(std=0.2)
    out, _ = m(inputs)
    assert out.shape == a.shape and not torch.equal(out, a)
    out.square().sum().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in m.parameters())
