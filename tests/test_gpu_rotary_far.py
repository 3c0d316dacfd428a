"""GPU test of rotary angles at far positions against angles reduced in 60 decimal digits."""
import decimal
import math

import pytest
import torch

from flashbev_b200 import rotary_axes

pytestmark = pytest.mark.gpu

PI = decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494459")


@pytest.mark.parametrize("base", [10000.0, 100.0])
@pytest.mark.parametrize("far", [1 << 12, 1 << 20, 1 << 24, 1 << 30, 1 << 40])
def test_angles_of_far_positions(cuda_device, far, base):
    pairs, L = 16, 40
    g = torch.Generator().manual_seed(far % 1000003)
    x = torch.randn(1, L, 1, 2 * pairs, generator=g)
    pos = (far + torch.randint(0, 1000, (L, 1), generator=g)) * torch.tensor([1, -1]).repeat(L // 2).view(L, 1)
    with decimal.localcontext() as ctx:
        ctx.prec = 60
        freq = [decimal.Decimal(base) ** (decimal.Decimal(-j) / pairs) for j in range(pairs)]
        angle = [[int(p) * f for f in freq] for p in pos.flatten()]
        left = torch.tensor([[float(a % (2 * PI)) for a in row] for row in angle], dtype=torch.float64)
        size = torch.tensor([[abs(float(a)) for a in row] for row in angle], dtype=torch.float64)
    a, b = x[0, :, 0, :pairs].double(), x[0, :, 0, pairs:].double()
    want = torch.cat([a * left.cos() - b * left.sin(), a * left.sin() + b * left.cos()], -1)
    # float64's part of an angle |angle| * 2^-49 (for base 10^4: (1 + ln(base) + 4) roundings of 2^-53 are less than 2^-49);
    # float32's: half a turn rounded (pi * 2^-25, doubled for sine and cosine), two products, a sum, the result
    tol = (a.abs() + b.abs()) * (size * 2.0 ** -49 + (math.pi + 5) * 2.0 ** -24)
    got = rotary_axes(x.to(cuda_device), pos.to(cuda_device), (pairs,), base=base).cpu()[0, :, 0].double()
    assert ((got - want).abs() <= torch.cat([tol, tol], -1)).all()
