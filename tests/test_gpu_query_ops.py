"""GPU tests of cross_attention, rotary_axes and add_rms_norm against plain float64 forms (tests/query_reference.py)."""
import math

import pytest
import torch

from flashbev_b200 import add_rms_norm, cross_attention, rotary_axes
from flashbev_b200.flash_bevpool import status_word
from tests import query_reference as R

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _rand(shape, dtype, seed, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    return torch.randn(*shape, generator=g, device=device).to(dtype)


def _run(q, k, v, dout, **kw):
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    out = cross_attention(q, k, v, **kw)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), dout)
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


def _compare(got, want, report=None, what=""):
    figures = {n: R.worst(got[n], want[n]) for n in got}
    if report:
        report(f"{what}: error / tolerance " + " ".join(f"{n} {x:.2f}" for n, x in figures.items()))
    assert all(x <= 1.0 for x in figures.values()), (what, figures)
    assert int(status_word(torch.device("cuda", 0)).item()) & 2 == 0


# (B, Lq, Lk, Hq, Hkv, D): one token to several tiles, odd sizes, shared heads, every width class
SHAPES = [
    (1, 1, 1, 1, 1, 64),
    (1, 1, 4224, 8, 2, 64),
    (3, 1, 1000, 8, 2, 128),
    (2, 5, 333, 6, 2, 64),
    (1, 16, 2500, 4, 1, 32),
    (2, 127, 129, 2, 2, 64),
    (1, 128, 128, 1, 1, 128),
    (1, 129, 255, 2, 1, 40),
    (1, 300, 700, 3, 3, 80),
    (2, 257, 640, 4, 2, 16),
    (1, 1000, 517, 2, 2, 96),
    (1, 43, 391, 15, 3, 8),
    (1, 260, 130, 7, 1, 128),
    (1, 70, 90, 2, 1, 33),
    (1, 33, 65, 2, 2, 1),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("masked", ["none", "lengths", "mask", "both"])
def test_attention_and_gradients(cuda_device, shape, dtype, masked):
    B, Lq, Lk, Hq, Hkv, D = shape
    q, k, v = _rand((B, Lq, Hq, D), dtype, 1), _rand((B, Lk, Hkv, D), dtype, 2), _rand((B, Lk, Hkv, D), dtype, 3)
    dout = _rand((B, Lq, Hq, D), dtype, 4)
    g = torch.Generator(device="cuda").manual_seed(5)
    lengths = torch.randint(0, Lk + 1, (B,), generator=g, device="cuda", dtype=torch.int32) if masked in ("lengths", "both") else None
    mask = torch.rand(B, Lk, generator=g, device="cuda") < 0.6 if masked in ("mask", "both") else None
    kw = {"key_lengths": lengths, "key_mask": mask}
    want = R.attention(q, k, v, R.allowed(B, Lk, lengths, mask), 1 / math.sqrt(D), dout)
    _compare(_run(q, k, v, dout, **kw), want, what=f"{shape} {dtype} {masked}")
    # the call without gradients gives the same
    assert R.worst(cross_attention(q, k, v, **kw), want["out"]) <= 1.0


# enough blocks that nothing is split: a block walks many tiles, the rings of tiles wrap
LONG = [(40, 1, 2500, 8, 4, 64), (40, 3, 1900, 4, 4, 128), (2, 1500, 2700, 16, 8, 64), (2, 1300, 2600, 8, 8, 128)]


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("shape", LONG, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("masked", ["none", "lengths", "mask", "both"])
def test_attention_of_many_tiles(cuda_device, shape, dtype, masked):
    B, Lq, Lk, Hq, Hkv, D = shape
    q, k, v = _rand((B, Lq, Hq, D), dtype, 1), _rand((B, Lk, Hkv, D), dtype, 2), _rand((B, Lk, Hkv, D), dtype, 3)
    dout = _rand((B, Lq, Hq, D), dtype, 4)
    g = torch.Generator(device="cuda").manual_seed(5)
    lengths = torch.randint(Lk // 2, Lk + 1, (B,), generator=g, device="cuda") if masked in ("lengths", "both") else None
    mask = torch.rand(B, Lk, generator=g, device="cuda") < 0.8 if masked in ("mask", "both") else None
    got = _run(q, k, v, dout, key_lengths=lengths, key_mask=mask)
    for b in range(0, B, 19):  # the float64 form sample by sample
        one = slice(b, b + 1)
        ok = R.allowed(1, Lk, None if lengths is None else lengths[one], None if mask is None else mask[one])
        _compare({n: t[one] for n, t in got.items()}, R.attention(q[one], k[one], v[one], ok, 1 / math.sqrt(D), dout[one]))


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("Lq", [1, 200])
def test_attention_ignores_what_may_not_be_attended(cuda_device, dtype, Lq):
    """NaN, infinities and the type's lowest value behind the length and in masked places change nothing, bit for bit."""
    B, Lk, H, D = 3, 500, 2, 64
    q, k, v = _rand((B, Lq, H, D), dtype, 1), _rand((B, Lk, H, D), dtype, 2), _rand((B, Lk, H, D), dtype, 3)
    dout = _rand((B, Lq, H, D), dtype, 4)
    lengths = torch.tensor([500, 130, 0], device="cuda", dtype=torch.int32)
    mask = torch.rand(B, Lk, generator=torch.Generator(device="cuda").manual_seed(6), device="cuda") < 0.7
    mask[0, 128:256] = False  # a whole tile of keys
    ok = R.allowed(B, Lk, lengths, mask)
    base = _run(q, k, v, dout, key_lengths=lengths, key_mask=mask)
    _compare(base, R.attention(q, k, v, ok, 1 / math.sqrt(D), dout))
    for bad in (math.nan, math.inf, -math.inf, torch.finfo(dtype).min):
        kb, vb = k.clone(), v.clone()
        kb[~ok], vb[~ok] = bad, bad
        got = _run(q, kb, vb, dout, key_lengths=lengths, key_mask=mask)
        for n in base:
            assert torch.equal(base[n], got[n]), (n, bad)
    assert not base["out"][2].any() and not base["dq"][2].any() and not base["dk"][~ok].any() and not base["dv"][~ok].any()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
def test_attention_empty_sizes(cuda_device, dtype):
    for B, Lq, Lk in ((0, 4, 5), (2, 0, 5), (2, 4, 0)):
        q, k = torch.ones(B, Lq, 4, 64, device="cuda", dtype=dtype), torch.ones(B, Lk, 2, 64, device="cuda", dtype=dtype)
        got = _run(q, k, k.clone(), torch.ones_like(q))
        for n, like in (("out", q), ("dq", q), ("dk", k), ("dv", k)):
            assert got[n].shape == like.shape and not got[n].any(), (B, Lq, Lk, n)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["fp32", "bf16", "fp16"])
def test_attention_large_scores(cuda_device, dtype):
    """Scores in the hundreds, rising along the keys: the running maximum moves in every tile, weights underflow."""
    B, Lq, Lk, H, D = 1, 150, 900, 2, 64
    q, k, v = _rand((B, Lq, H, D), dtype, 1), _rand((B, Lk, H, D), dtype, 2), _rand((B, Lk, H, D), dtype, 3)
    k = (k.float() * torch.linspace(0.1, 8, Lk, device="cuda").view(1, Lk, 1, 1)).to(dtype)
    q = (q.float() * 4).to(dtype)
    dout = _rand((B, Lq, H, D), dtype, 4)
    _compare(_run(q, k, v, dout), R.attention(q, k, v, R.allowed(B, Lk), 1 / math.sqrt(D), dout))
    _compare(_run(q, k, v, dout, scale=-0.3), R.attention(q, k, v, R.allowed(B, Lk), -0.3, dout))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
def test_attention_strided_and_shared_operands(cuda_device, dtype):
    """Keys and values as slices of one projection, heads in front of tokens, queries expanded over the batch, an odd offset."""
    B, Lq, Lk, H, D = 3, 140, 260, 4, 64
    kv = _rand((B, Lk, 2, H, D), dtype, 1)
    k, v = kv[:, :, 0], kv[:, :, 1]
    q = _rand((1, Lq, H, D), dtype, 2)
    dout = _rand((B, Lq, H, D), dtype, 3)
    want = R.attention(q.expand(B, -1, -1, -1), k, v, R.allowed(B, Lk), 1 / math.sqrt(D), dout)
    ql, kvl = q.clone().requires_grad_(), kv.clone().requires_grad_()
    out = cross_attention(ql.expand(B, -1, -1, -1), kvl[:, :, 0], kvl[:, :, 1])
    assert R.worst(out, want["out"]) <= 1.0
    dq, dkv = torch.autograd.grad(out, (ql, kvl), dout)
    u = R.unit(dtype)
    assert R.worst(dkv[:, :, 0], want["dk"]) <= 1.0 and R.worst(dkv[:, :, 1], want["dv"]) <= 1.0
    value, tol = want["dq"]
    total = value.sum(0, keepdim=True)
    assert R.worst(dq, (total, tol.sum(0, keepdim=True) + B * u * value.abs().sum(0, keepdim=True))) <= 1.0
    # the same values behind other strides
    alone = cross_attention(q.expand(B, -1, -1, -1), k, v)
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q.expand(B, -1, -1, -1), k, v)]
    assert torch.equal(alone, cross_attention(*heads_first))
    odd = torch.empty(k.numel() + 1, dtype=dtype, device="cuda")[1:].view(k.shape).copy_(k)
    assert torch.equal(alone, cross_attention(q.expand(B, -1, -1, -1), odd, v))
    one = k[:, :, :1].expand(-1, -1, H, -1)  # heads that repeat one head's keys
    assert R.worst(cross_attention(q.expand(B, -1, -1, -1), one, v),
                   R.attention(q.expand(B, -1, -1, -1), one, v, R.allowed(B, Lk), 1 / math.sqrt(D))["out"]) <= 1.0
    # an upstream gradient that is a broadcast view
    want_sum = R.attention(q.expand(B, -1, -1, -1), k, v, R.allowed(B, Lk), 1 / math.sqrt(D), torch.ones_like(dout))
    out = cross_attention(ql.expand(B, -1, -1, -1), kvl[:, :, 0], kvl[:, :, 1])
    assert R.worst(torch.autograd.grad(out.sum(), kvl)[0][:, :, 1], want_sum["dv"]) <= 1.0


def test_attention_offsets_beyond_32_bits(cuda_device):
    """Keys 4 MiB apart: the last ones lie beyond 2^32 elements."""
    step, Lk, D = 1 << 21, 2200, 64
    big = torch.empty(Lk * step, dtype=BF16, device="cuda")
    k = big.as_strided((1, Lk, 1, D), (0, step, D, 1), 0)
    v = big.as_strided((1, Lk, 1, D), (0, step, D, 1), D)
    k.copy_(_rand((1, Lk, 1, D), BF16, 1))
    v.copy_(_rand((1, Lk, 1, D), BF16, 2))
    for Lq in (1, 200):
        q, dout = _rand((1, Lq, 1, D), BF16, 3), _rand((1, Lq, 1, D), BF16, 4)
        _compare(_run(q, k, v, dout), R.attention(q, k, v, R.allowed(1, Lk), 1 / math.sqrt(D), dout))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("Lq", [3, 400])
def test_attention_is_the_same_from_run_to_run(cuda_device, dtype, Lq):
    q, k, v = _rand((2, Lq, 4, 64), dtype, 1), _rand((2, 1500, 2, 64), dtype, 2), _rand((2, 1500, 2, 64), dtype, 3)
    dout = _rand(q.shape, dtype, 4)
    a = _run(q, k, v, dout)
    for _ in range(3):
        b = _run(q, k, v, dout)
        assert all(torch.equal(a[n], b[n]) for n in a)


def test_attention_gradient_against_differences(cuda_device):
    """The gradient's product with a direction against central differences of the float64 form along it."""
    B, Lq, Lk, H, D = 2, 70, 150, 2, 32
    ts = [_rand((B, L, H, D), F32, i) for i, L in ((1, Lq), (2, Lk), (3, Lk))]
    dirs = [_rand(t.shape, F32, 10 + i) for i, t in enumerate(ts)]
    dout = _rand((B, Lq, H, D), F32, 4)
    ok, scale = R.allowed(B, Lk), 1 / math.sqrt(D)
    got = _run(*ts, dout)
    want = R.attention(*ts, ok, scale, dout)
    h = 1e-4
    for i, n in enumerate(("dq", "dk", "dv")):
        at = lambda sgn: [t.double() + sgn * h * dirs[i].double() if j == i else t.double() for j, t in enumerate(ts)]  # noqa: E731, B023
        f = lambda x: float((R_out(*x, ok, scale) * dout.double()).sum())  # noqa: E731, B023
        diff = (f(at(1)) - f(at(-1))) / (2 * h)
        along = float((got[n].double() * dirs[i].double()).sum())
        # the kernel's tolerance along the direction, and the difference's own error (h^2 and float64 rounding)
        tol = float((want[n][1] * dirs[i].double().abs()).sum()) + 1e-6 * (1 + abs(diff))
        assert abs(diff - along) <= tol, (n, diff, along, tol)


def R_out(q, k, v, ok, scale):
    qd, kd, vd = (t.transpose(1, 2) for t in (q, k, v))
    s = (qd @ kd.transpose(2, 3) * scale).masked_fill(~ok.view(ok.shape[0], 1, 1, -1), -math.inf)
    return (torch.softmax(s, -1) @ vd).transpose(1, 2)


@pytest.mark.parametrize("Lq", [1, 300])
def test_attention_on_streams_and_in_graphs(cuda_device, Lq):
    """Two streams at once, and two captured graphs replayed in turn and at once, give what the plain call gives."""
    sets = []
    for s in range(2):
        q, k, v = _rand((2, Lq, 4, 64), BF16, 10 * s + 1), _rand((2, 2000, 2, 64), BF16, 10 * s + 2), _rand((2, 2000, 2, 64), BF16, 10 * s + 3)
        sets.append((q, k, v, _rand(q.shape, BF16, 10 * s + 4)))
    want = [_run(*x) for x in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        got = []
        for st, x in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(_run(*x))
        torch.cuda.synchronize()
        assert all(torch.equal(w[n], g[n]) for w, g in zip(want, got) for n in w)
    graphs, held = [], []
    for x in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(_run(*x))
        graphs.append(graph)
    for _ in range(3):
        for h in held:
            for t in h.values():
                t.detach().zero_()
        torch.cuda.synchronize()
        for st, graph in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(w[n], h[n]) for w, h in zip(want, held) for n in w)


ROTARY = [  # B, L, H, D, sections
    (1, 1, 1, 2, (1,)),
    (1, 4224, 8, 64, (12, 10, 10)),
    (3, 37, 5, 80, (14, 13, 13)),
    (2, 100, 3, 32, (8, 8)),
    (2, 65, 2, 40, (5, 4, 3)),
    (1, 50, 1, 256, (64, 64)),
    (2, 33, 4, 18, (4, 0, 3)),
    (1, 700, 16, 128, (16, 24, 24)),
    (1, 9, 2, 10, (0, 0)),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("shape", ROTARY, ids=lambda s: "x".join(map(str, s[:4])))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("pos", ["float", "int32", "int64", "shared"])
def test_rotary(cuda_device, shape, dtype, interleaved, pos):
    B, L, H, D, sections = shape
    x, dout = _rand((B, L, H, D), dtype, 1).requires_grad_(), _rand((B, L, H, D), dtype, 2)
    g = torch.Generator(device="cuda").manual_seed(3)
    lead = (L,) if pos == "shared" else (B, L)
    if pos in ("float", "shared"):
        p = torch.randn(*lead, len(sections), generator=g, device="cuda") * 50
    else:
        p = torch.randint(-1000000, 1000000, (*lead, len(sections)), generator=g, device="cuda",
                          dtype=torch.int32 if pos == "int32" else torch.int64)
    out = rotary_axes(x, p, sections, interleaved=interleaved)
    assert out.is_contiguous() and out.dtype == dtype
    assert R.worst(out, R.rotary(x, p, sections, 10000.0, interleaved)) <= 1.0
    dx, = torch.autograd.grad(out, x, dout)
    assert R.worst(dx, R.rotary(dout, p, sections, 10000.0, interleaved, inverse=True)) <= 1.0
    rest = 2 * sum(sections)
    assert torch.equal(out[..., rest:], x[..., rest:])


def test_rotary_strided_and_far(cuda_device):
    x = _rand((2, 50, 3, 4, 64), BF16, 1)[:, :, 1]
    p = torch.arange(100, device="cuda", dtype=torch.int64).view(2, 50, 1) + (1 << 40)
    assert R.worst(rotary_axes(x, p, (32,)), R.rotary(x, p, (32,), 10000.0, False)) <= 1.0
    y = _rand((2, 4, 50, 64), F32, 2).transpose(1, 2)
    f = torch.full((50, 2), 3.0e6, device="cuda")
    for inter in (False, True):
        assert R.worst(rotary_axes(y, f, (10, 20), base=100.0, interleaved=inter), R.rotary(y, f, (10, 20), 100.0, inter)) <= 1.0
    odd = torch.empty(2 * 9 * 3 * 16 + 1, dtype=F16, device="cuda")[1:].view(2, 9, 3, 16).copy_(_rand((2, 9, 3, 16), F16, 3))
    q = torch.randn(9, 1, device="cuda")
    for inter in (False, True):
        assert R.worst(rotary_axes(odd, q, (8,), interleaved=inter), R.rotary(odd, q, (8,), 10000.0, inter)) <= 1.0
    # an expanded upstream gradient
    z = _rand((1, 4, 2, 16), F32, 4).requires_grad_()
    pz = torch.arange(4, device="cuda", dtype=torch.float32).view(4, 1)
    dz, = torch.autograd.grad(rotary_axes(z, pz, (8,), interleaved=True).sum(), z)
    assert R.worst(dz, R.rotary(torch.ones_like(z), pz, (8,), 10000.0, True, inverse=True)) <= 1.0
    assert rotary_axes(torch.empty(0, 4, 2, 16, device="cuda"), pz, (8,)).shape == (0, 4, 2, 16)
    assert rotary_axes(torch.empty(2, 4, 0, 16, device="cuda"), pz, (8,)).shape == (2, 4, 0, 16)


NORM = [(1, 256), (3, 1), (1000, 80), (37, 64), (5, 37), (6, 100), (700, 256), (9, 512), (3, 1000), (2, 2048), (5, 4096),
        (3, 8192), (2, 481), (2, 2041), (4, 4097), (2, 10000), (2, 8200)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("shape", NORM, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("form", ["full", "no_residual", "no_weight"])
def test_norm_and_gradients(cuda_device, shape, dtype, form):
    x = _rand(shape, dtype, 1).requires_grad_()
    r = None if form == "no_residual" else _rand(shape, dtype, 2).requires_grad_()
    w = None if form == "no_weight" else (1 + 0.2 * _rand(shape[-1:], F32, 3)).to(dtype).requires_grad_()
    dy, dh = _rand(shape, dtype, 4), _rand(shape, dtype, 5)
    y, h = add_rms_norm(x, r, w, eps=1e-5)
    want = R.norm(x, r, w, 1e-5, dy, None if r is None else dh)
    assert R.worst(y, want["y"]) <= 1.0 and R.worst(h, want["h"]) <= 1.0
    leaves = [t for t in (x, r, w) if t is not None]
    outs, ups = ((y,), (dy,)) if r is None else ((y, h), (dy, dh))
    grads = torch.autograd.grad(outs, leaves, ups, retain_graph=True)
    assert R.worst(grads[0], want["dx"]) <= 1.0
    if r is not None:
        assert torch.equal(grads[0], grads[1])
    if w is not None:
        assert R.worst(grads[-1], want["dw"]) <= 1.0
    # y alone, and the same gradients again
    only = R.norm(x, r, w, 1e-5, dy, None)
    assert R.worst(torch.autograd.grad(y, x, dy, retain_graph=True)[0], only["dx"]) <= 1.0
    again = torch.autograd.grad(outs, leaves, ups)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    with torch.no_grad():
        y2, h2 = add_rms_norm(x, r, w, eps=1e-5)
    assert torch.equal(y, y2) and torch.equal(h, h2)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("shape", NORM, ids=lambda s: "x".join(map(str, s)))
def test_norm_8bit(cuda_device, shape, dtype):
    x, r = _rand(shape, dtype, 1), _rand(shape, dtype, 2)
    w = (1 + 0.2 * _rand(shape[-1:], F32, 3)).to(dtype)
    x[0], r[0] = 0, 0  # a row of zeros
    q, scales, h = add_rms_norm(x, r, w, quantize=True)
    want = R.norm(x, r, w, 1e-6)
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape and scales.shape == x.shape[:-1]
    y, ytol = want["y"]
    top = y.abs().amax(-1)
    sc = torch.where(top > 0, top / 448, torch.ones_like(top))
    assert R.worst(scales, (sc, sc * (shape[-1] + 16) * 2.0 ** -24)) <= 1.0
    assert R.worst(h, want["h"]) <= 1.0
    # e4m3: half a step is 2^-4 of the value, 2^-10 below the smallest normal number 2^-6; y itself in float32
    back = q.double() * scales.double().unsqueeze(-1)
    u = R.unit(dtype)
    f32_tol = (ytol - u * y.abs()).clamp_min(0) + y.abs() * 2.0 ** -22
    assert R.worst(back, (y, (2.0 ** -4 * y.abs()).maximum(2.0 ** -10 * sc.unsqueeze(-1)) + 1.1 * f32_tol)) <= 1.0
    assert not q[0].double().any() and float(scales[0]) == 1.0


def test_norm_special_rows(cuda_device):
    x = _rand((4, 256), F32, 1)
    x[1, 7], x[2, 9] = math.nan, math.inf
    y, _ = add_rms_norm(x)
    assert torch.isnan(y[1]).all() and torch.isfinite(y[0]).all() and torch.isfinite(y[3]).all()
    q, s, _ = add_rms_norm(x, quantize=True)
    assert torch.isnan(s[1]) and torch.isfinite(s[0]) and torch.isfinite(s[3])
    assert add_rms_norm(torch.empty(0, 16, device="cuda"))[0].shape == (0, 16)
    w = torch.ones(16, device="cuda", requires_grad=True)
    y, _ = add_rms_norm(torch.empty(0, 16, device="cuda"), None, w)
    assert not torch.autograd.grad(y.sum(), w)[0].any()
    # the sum alone is used: its gradient passes through
    a, b = (_rand((3, 64), BF16, i).requires_grad_() for i in (1, 2))
    _, h = add_rms_norm(a, b)
    da, db = torch.autograd.grad(h, (a, b), torch.full_like(h, 2.0))
    assert (da == 2).all() and (db == 2).all()
    # strided rows and an odd address
    t = _rand((6, 2, 80), F16, 3)
    assert torch.equal(add_rms_norm(t[:, 0])[0], add_rms_norm(t[:, 0].contiguous())[0])
    odd = torch.empty(6 * 80 + 1, dtype=F16, device="cuda")[1:].view(6, 80).copy_(t[:, 0])
    assert R.worst(add_rms_norm(odd)[0], R.norm(odd, None, None, 1e-6)["y"]) <= 1.0
