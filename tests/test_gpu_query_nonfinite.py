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
