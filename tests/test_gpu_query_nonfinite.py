"""GPU tests of attention over values that are attended and not finite: NaN where the 64-bit form has it, whatever number of
blocks shares a row's keys, and every other row bit for bit what it is without them."""
import math

import pytest
import torch

from flashbev_b200 import cross_attention
from tests import query_reference as R

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["fp32", "bf16", "fp16"])


def _rand(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _run(q, k, v, dout, **kw):
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    out = cross_attention(q, k, v, **kw)
    return (out.detach(), *torch.autograd.grad(out, (q, k, v), dout))


def _same(a, b):
    return torch.equal(a.nan_to_num(nan=7.0, posinf=8.0, neginf=9.0), b.nan_to_num(nan=7.0, posinf=8.0, neginf=9.0))


@TYPES
@pytest.mark.parametrize("Lq,D", [(1, 64), (130, 64), (130, 128)])
def test_a_key_that_is_not_finite(cuda_device, Lq, D, dtype):
    """In every column of a tile, a sample each; the last two samples stay as they are."""
    B, Lk = 130, 200
    q, k, v = _rand((B, Lq, 2, D), dtype, 1), _rand((B, Lk, 1, D), dtype, 2), _rand((B, Lk, 1, D), dtype, 3)
    dout = _rand(q.shape, dtype, 4)
    base = _run(q, k, v, dout)
    b = torch.arange(128, device=cuda_device)
    for at in (b, Lk - 1 - b // 2):  # whole tiles, and the last one, which is not full
        kb = k.clone()
        kb[b, at, 0, 3] = math.nan
        for got, clean in zip(_run(q, kb, v, dout), base):
            assert torch.isnan(got[:128]).all() and torch.equal(got[128:], clean[128:])
        if dtype == F32:
            continue  # an infinity is NaN there
        kb[b, at, 0, 3] = math.inf
        out = cross_attention(q, kb, v)
        ok = R.allowed(B, Lk)
        ok[b, at] = False
        want, tol = R.attention(q, k, v, ok, 1 / math.sqrt(D))["out"]
        lost = q[..., 3] > 0  # a score of infinity; of -infinity where the query's number is negative
        lost[128:] = False
        assert torch.equal(torch.isnan(out), lost.unsqueeze(-1).expand_as(out)) and (q[..., 3] != 0).all()
        kept = ~lost
        kept[128:] = False
        assert R.worst(out[kept], (want[kept], tol[kept])) <= 1.0
        assert torch.equal(out[128:], base[0][128:])


# one query (both groups of a block share its keys, several blocks join), some, a grid whose last units are split; a width
# that takes the kernels of three parts, whose results are joined in 16 bits even when nothing is split
SIZES = [
    (1, 1, 4224, 8, 2, 64),
    (3, 1, 1000, 8, 2, 128),
    (2, 1, 1, 2, 2, 64),
    (40, 1, 700, 8, 4, 64),
    (1, 130, 2500, 4, 4, 64),
    (2, 130, 300, 4, 2, 40),
    (2, 300, 900, 2, 2, 96),
    (2, 70, 90, 4, 2, 33),
    (1, 2, 5000, 2, 1, 36),
    (1, 40000, 1100, 2, 2, 64),
]


@TYPES
@pytest.mark.parametrize("shape", SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("masked", ["none", "lengths", "mask"])
def test_a_query_that_is_not_finite(cuda_device, shape, masked, dtype):
    B, Lq, Lk, Hq, Hkv, D = shape
    q, k, v = _rand((B, Lq, Hq, D), dtype, 1), _rand((B, Lk, Hkv, D), dtype, 2), _rand((B, Lk, Hkv, D), dtype, 3)
    dout = _rand(q.shape, dtype, 4)
    lengths = mask = None
    if masked == "lengths":
        lengths = torch.tensor([max(Lk - 131 * b, 0) for b in range(B)], dtype=torch.int32, device=cuda_device)
    elif masked == "mask":
        mask = torch.rand(B, Lk, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda") < 0.6
        mask[-1] = False
    kw = {"key_lengths": lengths, "key_mask": mask}
    ok = R.allowed(B, Lk, lengths, mask)
    base = _run(q, k, v, dout, **kw)
    assert all(torch.isfinite(t).all() for t in base)
    bad = torch.zeros(B, Lq, Hq, dtype=torch.bool, device=cuda_device)
    bad[0, 0, 0] = bad[-1, Lq // 2, -1] = bad[0, -1, -1] = bad[B // 2, Lq // 3, 0] = True
    some = ok.any(1).view(B, 1, 1)                          # rows with keys
    head = (bad & some).any(1).view(B, Hkv, Hq // Hkv).any(2).unsqueeze(1)  # key heads that such a query reaches
    for value in (math.nan, math.inf, -math.inf):
        qb = q.clone()
        where = torch.nonzero(bad)
        qb[where[:, 0], where[:, 1], where[:, 2], D // 2] = value
        for b, i, h in where.tolist():  # the 64-bit form of these rows
            s = (k[b, ok[b], h // (Hq // Hkv)].double() @ qb[b, i, h].double()) / math.sqrt(D)
            assert s.numel() == 0 or torch.isnan(torch.softmax(s, 0)).all()
        out, dq, dk, dv = _run(qb, k, v, dout, **kw)
        for got, clean in ((out, base[0]), (dq, base[1])):
            assert torch.equal(torch.isnan(got), (bad & some).unsqueeze(-1).expand_as(got)), value
            assert torch.equal(got[~(bad & some)], clean[~(bad & some)]), value
        for got, clean in ((dk, base[2]), (dv, base[3])):
            lost = (head & ok.unsqueeze(-1)).unsqueeze(-1).expand_as(got)
            assert torch.equal(torch.isnan(got), lost), value
            assert torch.equal(got[~lost], clean[~lost]), value
        assert _same(cross_attention(qb, k, v, **kw), out)  # and without statistics


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("Lq,B,D", [(1, 1, 64), (1, 160, 64), (130, 1, 64), (130, 1, 128), (300, 70, 128)])
@pytest.mark.parametrize("Lk", [1000, 34000])
def test_scores_of_minus_infinity(cuda_device, Lk, Lq, B, D, dtype):
    """A row whose only key scores -infinity is no row without keys; beside another key it has no weight."""
    if B * Lk > 400000:
        B = max(B * 1000 // Lk, 1)
    q = (1 + _rand((B, Lq, 2, D), F32, 1).abs()).to(dtype)
    k, v = _rand((B, Lk, 1, D), dtype, 2), _rand((B, Lk, 1, D), dtype, 3)
    at, other = 2 * Lk // 3, Lk // 7
    k[:, at, 0, 5] = -math.inf
    mask = torch.zeros(B, Lk, dtype=torch.bool, device=cuda_device)
    mask[:, at] = True
    out, dq, dk, dv = _run(q, k, v, torch.ones_like(q), key_mask=mask)
    assert torch.isnan(out).all() and torch.isnan(dq).all()
    assert torch.equal(torch.isnan(dk[:, :, 0]).all(-1), mask) and torch.equal(torch.isnan(dv[:, :, 0]).all(-1), mask)
    assert not dk[~mask].any() and not dv[~mask].any()
    for near in (other, at + 1, at - 1):  # in another split, in the same tile
        both = mask.clone()
        both[:, near] = True
        # all the weight on one key: its values as they are
        assert torch.equal(cross_attention(q, k, v, key_mask=both), v[:, near:near + 1].expand(-1, Lq, 2, -1)), near


def test_scores_beyond_float32_are_not_zeros(cuda_device):
    """Products below float32's range are -infinity there: a row of only such keys shows it instead of looking unattended."""
    for Lq in (1, 200):
        for Lk in (1, 600):
            q, k = torch.full((2, Lq, 1, 64), 1e25, device=cuda_device), torch.full((2, Lk, 1, 64), -1e25, device=cuda_device)
            v = _rand((2, Lk, 1, 64), F32, 1)
            n = torch.tensor([Lk, 0], dtype=torch.int32, device=cuda_device)
            out = cross_attention(q, k, v, key_lengths=n)
            assert torch.isnan(out[0]).all() and not out[1].any()
