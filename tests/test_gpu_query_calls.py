"""GPU tests of how the query operators may be called: refusals, the same tensor twice, captured first calls, threads,
saved tensors that a hook moved, one gradient at a time."""
import math
import threading

import pytest
import torch

from flashbev_b200 import add_rms_norm, cross_attention, rotary_axes
from flashbev_b200.flash_bevpool import status_word
from tests import query_reference as R

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _rand(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def test_refusals(cuda_device):
    t = lambda *s, dtype=BF16: torch.zeros(*s, dtype=dtype, device=cuda_device)  # noqa: E731
    q, k = t(2, 3, 4, 16), t(2, 5, 2, 16)
    for args, kw in (
        ((q, k, t(2, 6, 2, 16)), {}),                       # values of another length
        ((q, t(1, 5, 2, 16), t(1, 5, 2, 16)), {}),          # another batch
        ((q, t(2, 5, 3, 16), t(2, 5, 3, 16)), {}),          # heads that do not divide
        ((q, t(2, 5, 0, 16), t(2, 5, 0, 16)), {}),
        ((q, t(2, 5, 2, 8), t(2, 5, 2, 8)), {}),            # another width
        ((t(2, 3, 4, 136), t(2, 5, 2, 136), t(2, 5, 2, 136)), {}),
        ((q[0], k[0], k[0]), {}),
        ((q, k.float(), k.float()), {}),
        ((q, k, k.half()), {}),
        ((q.double(), k.double(), k.double()), {}),
        ((q, k, k), {"scale": math.nan}),
        ((q, k, k), {"scale": math.inf}),
        ((q, k, k), {"scale": -2e30}),
        ((q, k, k), {"key_lengths": t(2, dtype=F32)}),
        ((q, k, k), {"key_lengths": t(3, dtype=torch.int32)}),
        ((q, k, k), {"key_mask": t(2, 5, dtype=torch.uint8)}),
        ((q, k, k), {"key_mask": t(2, 6, dtype=torch.bool)}),
        ((q, k, k), {"key_mask": t(2, dtype=torch.bool)}),
    ):
        with pytest.raises(ValueError):
            cross_attention(*args, **kw)
    with pytest.raises(RuntimeError, match="CUDA"):
        cross_attention(q, k.cpu(), k.cpu())
    p = t(3, 2, dtype=F32)
    for x, pos, sections, kw in (
        (q, p, (4, 5), {}),                                 # more pairs than the head has
        (q, p, (4,), {}),
        (q, p, (4, -1), {}),
        (q, p, (4, 2.0), {}),
        (q, p, (), {}),
        (q, t(3, 2, dtype=F16), (4, 4), {}),
        (q, t(4, 2, dtype=F32), (4, 4), {}),
        (q, t(1, 3, 2, dtype=F32), (4, 4), {}),
        (q, p.cpu(), (4, 4), {}),
        (q, p, (4, 4), {"base": 0.0}),
        (q, p, (4, 4), {"base": math.nan}),
        (q, p.clone().requires_grad_(), (4, 4), {}),
        (t(2, 3, 4, 258), p, (4, 4), {}),
        (t(2, 3, 4, 15), p, (3, 4), {"interleaved": True}),
        (q[0], p, (4, 4), {}),
    ):
        with pytest.raises(ValueError):
            rotary_axes(x, pos, sections, **kw)
    x, w = t(4, 16), t(16)
    for args, kw in (
        ((x, t(4, 8)), {}), ((x, t(4, 16, dtype=F32)), {}), ((x, None, t(8)), {}), ((x, None, t(4, 16)), {}), ((t(4, 0),), {}),
        ((t(()),), {}), ((x,), {"eps": -1.0}), ((x,), {"eps": math.nan}), ((x,), {"eps": math.inf}),
        ((x, None, w.requires_grad_()), {"quantize": True}),
    ):
        with pytest.raises(ValueError):
            add_rms_norm(*args, **kw)
    # nothing of the above left a call behind: the next ones are right
    assert not cross_attention(q, k, k).any()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
def test_the_same_tensor_twice(cuda_device, dtype):
    """Keys that are the values too, and queries that are both: the gradients add up."""
    x = _rand((2, 150, 2, 64), dtype, 1).requires_grad_()
    dout = _rand(x.shape, dtype, 2)
    want = R.attention(x, x, x, R.allowed(2, 150), 0.125, dout)
    out = cross_attention(x, x, x)
    assert R.worst(out, want["out"]) <= 1.0
    dx, = torch.autograd.grad(out, x, dout)
    parts = [want[n] for n in ("dq", "dk", "dv")]
    total = sum(v for v, _ in parts)
    u = R.unit(dtype)  # the two additions round as well
    size = sum(v.abs() for v, _ in parts)
    assert R.worst(dx, (total, sum(e for _, e in parts) + 2 * u * size)) <= 1.0
    y = _rand((7, 80), dtype, 3).requires_grad_()
    n, h = add_rms_norm(y, y)
    assert torch.equal(h, y + y)
    g, = torch.autograd.grad(h, y, torch.ones_like(h))
    assert (g == 2).all()


def test_norm_without_residual_returns_its_argument(cuda_device):
    x = _rand((6, 2, 80), F16, 3)[:, 0]  # not contiguous
    assert add_rms_norm(x)[1] is x
    assert add_rms_norm(x, quantize=True)[2] is x


def test_strides_of_dimensions_of_one(cuda_device):
    """A head cut out of an odd row: the strides of dimensions of one are odd, and not used."""
    for dtype in (F32, BF16):
        x, p = _rand((1, 1, 1, 17), dtype, 1)[..., :16], torch.full((1, 1), 3.0, device=cuda_device)
        for inter in (False, True):
            assert R.worst(rotary_axes(x, p, (8,), interleaved=inter), R.rotary(x, p, (8,), 10000.0, inter)) <= 1.0
        k = _rand((1, 40, 1, 17), dtype, 2)[..., :16]
        assert R.worst(cross_attention(x, k, k), R.attention(x, k, k, R.allowed(1, 40), 0.25)["out"]) <= 1.0


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
def test_one_gradient_at_a_time(cuda_device, dtype):
    q, k, v = _rand((2, 200, 4, 64), dtype, 1), _rand((2, 900, 2, 64), dtype, 2), _rand((2, 900, 2, 64), dtype, 3)
    dout = _rand(q.shape, dtype, 4)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    every = torch.autograd.grad(cross_attention(*leaves), leaves, dout)
    for i in range(3):
        args = [q, k, v]
        args[i] = leaves[i]
        one, = torch.autograd.grad(cross_attention(*args), leaves[i], dout)
        assert torch.equal(one, every[i]), i


def test_saved_tensors_that_a_hook_moved(cuda_device):
    q, k, v = (_rand((2, L, 2, 64), BF16, i).requires_grad_() for i, L in ((1, 70), (2, 300), (3, 300)))
    mask = torch.arange(300, device=cuda_device) % 3 > 0
    dout = _rand(q.shape, BF16, 4)
    x, w = _rand((9, 80), BF16, 5).requires_grad_(), _rand((80,), BF16, 6).requires_grad_()

    def step():
        out = cross_attention(q, k, v, key_mask=mask)
        y, _ = add_rms_norm(x, None, w)
        return out, y

    def grads(out, y):
        return [*torch.autograd.grad(out, (q, k, v), dout), *torch.autograd.grad(y, (x, w), torch.ones_like(y))]

    want = grads(*step())
    with torch.autograd.graph.save_on_cpu():
        held = step()
    assert all(torch.equal(a, b) for a, b in zip(grads(*held), want))


def test_first_call_is_captured(cuda_device):
    """Sizes no other call has: the plan, the kernels' attributes and the workspace are made while a graph is captured."""
    q, k = _rand((1, 131, 6, 56), BF16, 1), _rand((1, 1777, 3, 56), BF16, 2)
    p = torch.arange(131, device=cuda_device, dtype=F32).view(-1, 1)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        turned = rotary_axes(q, p, (28,))
        out = cross_attention(turned, k, k)
        y, scales, h = add_rms_norm(out.flatten(2), q.flatten(2), quantize=True)
    for _ in range(2):
        for t in (turned, out, scales, h):
            t.zero_()
        graph.replay()
    torch.cuda.synchronize()
    plain = cross_attention(rotary_axes(q, p, (28,)), k, k)
    assert torch.equal(out, plain)
    again = add_rms_norm(plain.flatten(2), q.flatten(2), quantize=True)
    assert torch.equal(scales, again[1]) and torch.equal(h, again[2]) and torch.equal(y.view(torch.uint8), again[0].view(torch.uint8))


def test_rotary_and_norm_in_graphs_with_gradients(cuda_device):
    x = _rand((2, 90, 3, 32), F32, 1).requires_grad_()
    r, w = _rand((2, 90, 96), F32, 2).requires_grad_(), _rand((96,), F32, 3).requires_grad_()
    p = torch.randint(-500, 500, (2, 90, 2), device=cuda_device)

    def step():
        y, h = add_rms_norm(rotary_axes(x, p, (8, 8)).flatten(2), r, w)
        return [t.detach() for t in (y, h, *torch.autograd.grad(y.sum() + h.sum(), (x, r, w)))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(2):
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_threads_on_streams_of_their_own(cuda_device):
    sets, want, wrong = [], [], []
    for i in range(3):
        q, k = _rand((2, 3 + 60 * i, 4, 64), BF16, 2 * i), _rand((2, 1200, 2, 64), BF16, 2 * i + 1)
        sets.append((q, k))
        want.append((cross_attention(q, k, k), add_rms_norm(q)[0]))
    torch.cuda.synchronize()

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(30):
                    q, k = sets[i]
                    got = cross_attention(q, k, k), add_rms_norm(q)[0]
                torch.cuda.current_stream().synchronize()
            if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                wrong.append(i)
        except Exception as e:  # noqa: BLE001  reported by the test, not lost in the thread
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong


def _holes(B, Lk, seed):
    """Masks with runs of any length taken away, and within what is left single keys; the last sample keeps three keys, the
    first none."""
    g = torch.Generator().manual_seed(seed)
    mask = torch.rand(B, Lk, generator=g) < 0.9
    for b in range(B):
        for _ in range(3):
            at = int(torch.randint(0, Lk, (1,), generator=g))
            mask[b, at:at + int(torch.randint(1, max(Lk // 2, 2), (1,), generator=g))] = False
    if B > 1:
        mask[-1] = False
        mask[-1, Lk // 2:Lk // 2 + 3] = True
        mask[0] = False
    return mask.cuda()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("lengths", [False, True])
@pytest.mark.parametrize("shape", [(4, 300, 2000, 4, 2, 64), (3, 1, 3001, 8, 2, 128), (3, 260, 1500, 2, 2, 96), (5, 3, 700, 4, 1, 32)],
                         ids=lambda s: "x".join(map(str, s)))
def test_masks_that_empty_whole_tiles(cuda_device, shape, lengths, dtype):
    B, Lq, Lk, Hq, Hkv, D = shape
    q, k, v = _rand((B, Lq, Hq, D), dtype, 1), _rand((B, Lk, Hkv, D), dtype, 2), _rand((B, Lk, Hkv, D), dtype, 3)
    dout, mask = _rand(q.shape, dtype, 4), _holes(B, Lk, 5)
    n = torch.tensor([Lk - 129 * b for b in range(B)], dtype=torch.int32, device=cuda_device) if lengths else None
    ok = R.allowed(B, Lk, n, mask)
    want = R.attention(q, k, v, ok, 1 / math.sqrt(D), dout)
    k[~ok], v[~ok] = math.nan, math.nan
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = cross_attention(*leaves, key_lengths=n, key_mask=mask)
    assert R.worst(out, want["out"]) <= 1.0
    for name, got in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, dout)):
        assert R.worst(got, want[name]) <= 1.0, name


def test_more_masked_tiles_than_a_block_lists(cuda_device):
    B, Lk = 74, 34000
    q, k = _rand((B, 1, 4, 64), BF16, 1), _rand((B, Lk, 2, 64), BF16, 2)
    mask = _holes(B, Lk, 3)
    out = cross_attention(q, k, k, key_mask=mask)
    for b in (0, 1, 40, 73):
        one = slice(b, b + 1)
        want = R.attention(q[one], k[one], k[one], R.allowed(1, Lk, None, mask[one]), 0.125, None)
        assert R.worst(out[one], want["out"]) <= 1.0, b


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Lq", [1, 100, 128, 129, 300, 640])
def test_maximum_that_rises_late(cuda_device, Lq, D, dtype):
    """Every number of row tiles a block may have, with scores that rise along the keys, so that the output so far is
    rescaled in late tiles, and with first tiles that are masked."""
    Lk = 1100
    q, k, v = _rand((1, Lq, 2, D), dtype, 1), _rand((1, Lk, 2, D), dtype, 2), _rand((1, Lk, 2, D), dtype, 3)
    k = (k.float() * torch.linspace(0.05, 6, Lk, device=cuda_device).view(1, Lk, 1, 1)).to(dtype)
    q, dout = (q.float() * 4).to(dtype), _rand(q.shape, dtype, 4)
    for first in (0, 1, 200, 520):
        mask = torch.arange(Lk, device=cuda_device) >= first
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        out = cross_attention(*leaves, key_mask=mask)
        want = R.attention(q, k, v, R.allowed(1, Lk, None, mask), 1 / math.sqrt(D), dout)
        assert R.worst(out, want["out"]) <= 1.0, first
        for name, got in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, dout)):
            assert R.worst(got, want[name]) <= 1.0, (first, name)
    assert int(status_word(torch.device("cuda", 0)).item()) & 2 == 0
