"""Plain float64 forms of the query operators and, for each result, how far a correct kernel may be from it.

Every tolerance is element-wise and counts roundings.  u is half a step of the tensor's type (torch.finfo(t).eps / 2);
a sum of n float32 products is off by at most n * 2^-24 times the sum of their absolute values, doubled here for the
order and split of the sum.  For 16-bit inputs the attention kernels round two intermediates to that type, the softmax
weights and the score gradients: one u each of the magnitudes they multiply, and 2^-25 where float16 has no finer step.
A weight below 2^-126, float32's and bfloat16's smallest normal number, may become zero: 2^-126 absolute.
The rounding of a result is u of its magnitude down to the type's smallest normal number; below it the steps stay as wide
as there (float16: 2^-24 below 2^-14), so it is never less than half of that step: 2^-14 * 2^-11 = 2^-25 for float16.
"""
import math

import torch


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def last(value, dtype):
    """Rounding of the result `value` to dtype: half a step, u of the value but no less than u of the smallest normal."""
    return unit(dtype) * value.abs().clamp_min(torch.finfo(dtype).tiny)


def allowed(B, Lk, lengths=None, mask=None, device="cuda"):
    ok = torch.ones(B, Lk, dtype=torch.bool, device=device)
    if lengths is not None:
        ok &= torch.arange(Lk, device=device).view(1, -1) < lengths.to(device).view(-1, 1)
    if mask is not None:
        ok &= mask.to(device)
    return ok


def _heads(x, group=1):
    x = x.detach().double().transpose(1, 2)
    return x.repeat_interleave(group, dim=1)


def attention(q, k, v, ok, scale, dout=None):
    """{name: (value, tolerance)} of out and, with dout, dq, dk, dv, in float64 and the tensors' layouts."""
    B, Lq, Hq, D = q.shape
    Lk, Hkv = k.shape[1], k.shape[2]
    G, dt = Hq // Hkv, q.dtype
    u = unit(dt)
    low = dt != torch.float32
    # exponentials: 2^-21 relative (two float32 units of 2^x and its argument's rounding), 2^-12 where the weight is
    # rounded to 16 bits anyway
    e = 2.0 ** -12 if low else 2.0 ** -20
    ui = u if low else 2.0 ** -21          # rounding of the weights before they meet the values
    sub = 2.0 ** -25 if dt == torch.float16 else 2.0 ** -126
    f32 = 2.0 ** -23
    qd, kd, vd = _heads(q), _heads(k, G), _heads(v, G)
    bar = ok.view(B, 1, 1, Lk)
    kd, vd = (torch.where(ok.view(B, 1, Lk, 1), x, torch.zeros_like(x)) for x in (kd, vd))
    s = (qd @ kd.transpose(2, 3)) * scale
    s = s.masked_fill(~bar, -math.inf)
    m = s.amax(-1, keepdim=True) if Lk else s.new_full((*s.shape[:3], 1), -math.inf)
    p = torch.exp(s - m.clamp_min(-1e300))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    out = p @ vd
    # relative error of a weight from its score: both the score and the row's statistics carry it
    es = (qd.abs() @ kd.abs().transpose(2, 3)) * abs(scale) * (D + 8) * f32
    es = es.masked_fill(~bar, 0.0)
    dp_rel = es + es.amax(-1, keepdim=True) if Lk else es
    rel = 2 * e + dp_rel + Lk * 2.0 ** -24
    back = lambda x: x.transpose(1, 2)  # noqa: E731
    fold = lambda x: back(x.view(B, Hkv, G, Lk, D).sum(2))  # noqa: E731
    out_tol = last(out, dt) + (p * (ui + rel)) @ vd.abs() + Lk * f32 * (p @ vd.abs()) + sub * vd.abs().sum(2, keepdim=True)
    res = {"out": (back(out), back(out_tol))}
    if dout is None:
        return res
    g = _heads(dout)
    n = Lq * G
    dv = p.transpose(2, 3) @ g
    dv_tol = (p * (ui + rel)).transpose(2, 3) @ g.abs() + n * f32 * (p.transpose(2, 3) @ g.abs()) + sub * g.abs().sum(2, keepdim=True)
    dp = g @ vd.transpose(2, 3)
    delta = (g * out).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    # dp in float32; delta from the rounded output, whose own error counts too
    dp_abs = D * f32 * (g.abs() @ vd.abs().transpose(2, 3))
    delta_abs = (g.abs() * out_tol).sum(-1, keepdim=True) + D * f32 * (g.abs() * out.abs()).sum(-1, keepdim=True)
    ds_tol = ds.abs() * (ui + rel) + p * (1 + rel) * (dp_abs + delta_abs) + sub * (1 + (dp - delta).abs()) * bar
    dq = (ds @ kd) * scale
    dq_tol = last(dq, dt) + abs(scale) * (ds_tol @ kd.abs() + Lk * f32 * (ds.abs() @ kd.abs()))
    dk = (ds.transpose(2, 3) @ qd) * scale
    dk_tol = abs(scale) * (ds_tol.transpose(2, 3) @ qd.abs() + n * f32 * (ds.abs().transpose(2, 3) @ qd.abs()))
    dk, dv, dk_tol, dv_tol = fold(dk), fold(dv), fold(dk_tol), fold(dv_tol)
    res["dq"] = (back(dq), back(dq_tol))
    res["dk"] = (dk, dk_tol + last(dk, dt))
    res["dv"] = (dv, dv_tol + last(dv, dt))
    return res


def rotary(x, positions, sections, base, interleaved, inverse=False):
    """(value, tolerance).  Angle: float64 up to one rounding of the remaining half turn to float32 (pi * 2^-25, doubled for
    the sine's own error), then two products and a sum in float32 and the rounding of the result."""
    P = sum(sections)
    axis = [a for a, s in enumerate(sections) for _ in range(s)]
    freq = torch.tensor([base ** (-j / s) for s in sections for j in range(s)], dtype=torch.float64, device=x.device)
    pos = positions.double() if positions.dim() == 3 else positions.double().unsqueeze(0)
    ang = (pos[..., axis] * freq).unsqueeze(2)
    c, s = torch.cos(ang), torch.sin(ang) * (-1 if inverse else 1)
    z = x.detach().double()
    y, tol = z.clone(), torch.zeros_like(z)
    i0 = torch.arange(P, device=x.device) * 2 if interleaved else torch.arange(P, device=x.device)
    i1 = i0 + 1 if interleaved else i0 + P
    a, b = z[..., i0], z[..., i1]
    y[..., i0], y[..., i1] = a * c - b * s, a * s + b * c
    # float64 positions times frequencies: half a step of the product is an angle's error here as well
    err = (a.abs() + b.abs()) * (math.pi * 2.0 ** -24 + 4 * 2.0 ** -24 + ang.abs() * 2.0 ** -50)
    tol[..., i0], tol[..., i1] = err, err
    return y, tol + last(y, x.dtype)


def norm(x, residual, weight, eps, dy=None, dh=None):
    """{name: (value, tolerance)} of y, h and, with dy / dh, dx and dw."""
    C, dt = x.shape[-1], x.dtype
    u, f32 = unit(dt), 2.0 ** -24
    xd, w = x.detach().double(), torch.ones(C, dtype=torch.float64, device=x.device) if weight is None else weight.detach().double()
    h = xd + (0 if residual is None else residual.detach().double())
    s = (h.square().mean(-1, keepdim=True) + eps).rsqrt()
    n = h * s
    y = n * w
    # a positive sum of C squares, a root, a quotient, three products: relative
    rel = (C + 12) * f32
    res = {"y": (y, last(y, dt) + rel * y.abs()), "h": (h, last(h, dt) + f32 * h.abs()), "rstd": (s, rel * s)}
    if dy is None and dh is None:
        return res
    zero = torch.zeros_like(h)
    g = zero if dy is None else dy.detach().double() * w
    d = zero if dh is None else dh.detach().double()
    dot = (g * n).mean(-1, keepdim=True)
    dx = d + s * (g - n * dot)
    uh = u + f32 if residual is not None else 0.0  # h is re-read rounded
    n_tol = n.abs() * (uh + rel)
    dot_tol = (g.abs() * n_tol).mean(-1, keepdim=True) + (C + 4) * f32 * (g * n).abs().mean(-1, keepdim=True)
    dx_tol = last(dx, dt) + s * (n_tol * dot.abs() + n.abs() * dot_tol + (rel + 4 * f32) * (g.abs() + (n * dot).abs())) + 2 * f32 * d.abs()
    res["dx"] = (dx, dx_tol)
    if dy is not None:
        t = dy.detach().double()
        rows = n.numel() // C
        dw = (t * n).reshape(-1, C).sum(0)
        dw_tol = last(dw, dt) + (t.abs() * n_tol).reshape(-1, C).sum(0) + (rows + 4) * f32 * (t * n).abs().reshape(-1, C).sum(0)
        res["dw"] = (dw, dw_tol)
    return res


def worst(got, want):
    """Largest error in units of the tolerance; not finite where one side is and the other is not."""
    value, tol = want
    got = got.detach().double()
    assert got.shape == value.shape, (got.shape, value.shape)
    if got.numel() == 0:
        return 0.0
    if not torch.isfinite(got).all():
        return math.inf
    return float(((got - value).abs() / tol.expand_as(value).clamp_min(1e-300)).max())
