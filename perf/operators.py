"""Cases of the operators that attend from BEV queries to camera tokens: what is timed, and what it is compared with.

Three operators stand next to the pooling operator, for the view transform in which BEV cells ask the cameras' tokens
instead of sampling them:

  cross_attention  queries [B,Lq,Hq,D] over the camera tokens' keys and values [B,Lk,Hkv,D] (Hq a multiple of Hkv),
                   with a number of valid tokens for each sample and / or a mask over its tokens;
  rotary_axes      rotary positions with several axes (time, height, width of a token; y, x of a BEV cell);
  add_rms_norm     the residual's addition and the root-mean-square norm of the sum, optionally with an output in
                   8 bits and a scale for each row.

``run`` is their plain form in elementary torch operations, or, with ``own`` set, the calls of ``flashbev_b200``.
"""
import math

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_E4M3_MAX = 448.0


def listed():
    att = {"op": "cross_attention"}
    rot = {"op": "rotary_axes"}
    nrm = {"op": "add_rms_norm"}
    return [
        # one query token over the tokens of six 16 x 44 cameras: the smallest serving call, where latency counts
        {"name": "attention_one_query_bf16", **att, "dtype": "bf16", "B": 1, "Lq": 1, "Lk": 4224, "Hq": 8, "Hkv": 2, "D": 64,
         "mask": "none", "train": False},
        # one query token for each of 64 samples over six 32 x 88 cameras, padded to the longest sample: bound by the bytes
        # of keys and values
        {"name": "attention_one_query_batch_fp16", **att, "dtype": "fp16", "B": 64, "Lq": 1, "Lk": 16896, "Hq": 8, "Hkv": 2,
         "D": 128, "mask": "lengths", "train": False},
        # some hundred object queries, odd sizes, one camera of each sample missing
        {"name": "attention_objects_bf16", **att, "dtype": "bf16", "B": 4, "Lq": 901, "Lk": 4219, "Hq": 8, "Hkv": 8, "D": 32,
         "mask": "camera", "train": False},
        # every cell of the 200 x 200 grid over six 16 x 44 cameras: the ordinary inference call
        {"name": "attention_grid_bf16", **att, "dtype": "bf16", "B": 1, "Lq": 40000, "Lk": 4224, "Hq": 4, "Hkv": 4, "D": 64,
         "mask": "none", "train": False},
        # the 128 x 128 grid over six 32 x 88 cameras with wide heads: the largest
        {"name": "attention_grid_wide_fp16", **att, "dtype": "fp16", "B": 1, "Lq": 16384, "Lk": 16896, "Hq": 4, "Hkv": 4, "D": 128,
         "mask": "none", "train": False},
        # a training step: output and the gradients of queries, keys and values, keys shared by two heads, padded batch
        {"name": "attention_train_bf16", **att, "dtype": "bf16", "B": 2, "Lq": 10000, "Lk": 4224, "Hq": 8, "Hkv": 4, "D": 64,
         "mask": "lengths", "train": True},
        # the same in 32 bits on a small grid, head width of the 80-channel features
        {"name": "attention_train_fp32", **att, "dtype": "fp32", "B": 1, "Lq": 2500, "Lk": 1056, "Hq": 4, "Hkv": 4, "D": 80,
         "mask": "none", "train": True},
        # positions (frame, row, column) of the tokens of six 16 x 44 cameras, frames counted from far
        {"name": "rotary_tokens_bf16", **rot, "dtype": "bf16", "B": 1, "L": 4224, "H": 8, "D": 64, "axes": 3, "far": 100000,
         "interleaved": False, "train": False},
        # positions (y, x) in metres of the cells of a 200 x 200 grid, four samples, with the gradient
        {"name": "rotary_grid_fp32_train", **rot, "dtype": "fp32", "B": 4, "L": 40000, "H": 8, "D": 32, "axes": 2, "far": 0,
         "interleaved": True, "train": True},
        # the residual stream of a 200 x 200 grid in 256 channels, four samples: output, sum and all gradients
        {"name": "norm_grid_bf16_train", **nrm, "dtype": "bf16", "rows": 160000, "C": 256, "quantize": False, "train": True},
        # the same stream in 80 channels, serving, output in 8 bits with a scale for each row
        {"name": "norm_grid_fp16_8bit", **nrm, "dtype": "fp16", "rows": 40000, "C": 80, "quantize": True, "train": False},
        # one token in 32 bits: latency
        {"name": "norm_one_token_fp32", **nrm, "dtype": "fp32", "rows": 1, "C": 256, "quantize": False, "train": False},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["cross_attention", "cross_attention", "rotary_axes", "add_rms_norm"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "cross_attention":
        train = rng.random() < 0.4
        D = rng.choice([16, 32, 40, 64, 64, 80, 96, 128])
        Hkv = rng.choice([1, 2, 4, 8])
        Hq = Hkv * rng.choice([1, 1, 2, 4])
        few = rng.random() < 0.35
        B = _spread(rng, 1, 64) if few else rng.randint(1, 4)
        Lq = rng.choice([1, 1, 2, rng.randint(3, 16)]) if few else _spread(rng, 17, 40000)
        # a gradient through a softmax over a single key is zero but for rounding: training has some tens of tokens
        Lk = _spread(rng, 32 if train else 1, 16896)
        most = 1e9 if dtype == "fp32" else (4e10 if train else 1.2e11)  # products of a query's and a key's numbers
        while B * Hq * Lq * Lk * D > most:
            if Lq > 1 and (Lk < 2000 or rng.random() < 0.5):
                Lq = Lq * 2 // 3
            else:
                Lk = Lk * 2 // 3 + 1
        return {"op": op, "dtype": dtype, "B": B, "Lq": Lq, "Lk": Lk, "Hq": Hq, "Hkv": Hkv, "D": D,
                "mask": rng.choice(["none", "lengths", "camera"]), "train": train}
    if op == "rotary_axes":
        D, H = rng.choice([16, 32, 64, 80, 128]), rng.choice([1, 2, 4, 8, 16])
        L, B = _spread(rng, 1, 40000), rng.randint(1, 4)
        while B * L * H * D > 4 * 40000 * 8 * 32:
            L = L * 2 // 3
        return {"op": op, "dtype": dtype, "B": B, "L": L, "H": H, "D": D, "axes": rng.choice([1, 2, 3]),
                "far": rng.choice([0, 0, 1000, 100000, 1000000]), "interleaved": rng.random() < 0.5, "train": rng.random() < 0.5}
    C = rng.choice([64, 80, 256, 256, 1000, 2048, 37, rng.randint(8, 4096)])
    rows = max(1, _spread(rng, 1, 160000) * 256 // max(C, 256))
    quantize = rng.random() < 0.4
    return {"op": op, "dtype": dtype, "rows": rows, "C": C, "quantize": quantize,
            "train": not quantize and rng.random() < 0.6}


def _sections(case):
    """How many of the D / 2 rotated pairs go to each axis: even shares, the first axis takes what is left over last."""
    pairs, axes = case["D"] // 2, case["axes"]
    share = pairs // axes
    return [pairs - share * (axes - 1)] + [share] * (axes - 1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    t = _TYPES[case["dtype"]]
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=torch.float32).to(t)  # noqa: E731
    state = {"case": case}
    if case["op"] == "cross_attention":
        B, Lq, Lk, Hq, Hkv, D = (case[n] for n in ("B", "Lq", "Lk", "Hq", "Hkv", "D"))
        # queries a little longer than unit variance: some keys stand out of the softmax, as in a trained model
        state["q"] = (rand(B, Lq, Hq, D).float() * 1.5).to(t)
        state["k"], state["v"] = rand(B, Lk, Hkv, D), rand(B, Lk, Hkv, D)
        state["lengths"] = state["mask"] = None
        if case["mask"] == "lengths":
            # the samples' encoders gave between half of the longest and all of it
            state["lengths"] = torch.randint((Lk + 1) // 2, Lk + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        elif case["mask"] == "camera":
            # one of six cameras is missing in each sample
            lost = torch.randint(0, 6, (B, 1), generator=g, device="cuda")
            state["mask"] = (torch.arange(Lk, device="cuda") * 6 // Lk).view(1, Lk) != lost
        if case["train"]:
            state["dout"] = rand(B, Lq, Hq, D)
            for n in ("q", "k", "v"):
                state[n].requires_grad_()
    elif case["op"] == "rotary_axes":
        B, L, H, D = (case[n] for n in ("B", "L", "H", "D"))
        state["x"] = rand(B, L, H, D)
        at = torch.arange(L, device="cuda")
        side = max(1, math.isqrt(L))
        if case["axes"] == 3:
            # six cameras' tokens: frame, row, column
            per = -(-L // 6)
            pos = [at // per, at % per // 44, at % per % 44]
        elif case["axes"] == 2:
            # metres from the vehicle
            pos = [(at // side - side // 2) * 0.5, (at % side - side // 2) * 0.5]
        else:
            pos = [at]
        pos = torch.stack([p.to(torch.float32) for p in pos], dim=-1)
        pos[:, 0] += case["far"]
        if B > 1:
            # each sample from a place of its own
            pos = pos.unsqueeze(0) + torch.randint(0, 100, (B, 1, case["axes"]), generator=g, device="cuda").float()
        state["positions"] = pos.contiguous()
        if case["train"]:
            state["dout"] = rand(B, L, H, D)
            state["x"].requires_grad_()
    else:
        rows, C = case["rows"], case["C"]
        state["x"], state["residual"] = rand(rows, C), rand(rows, C)
        state["weight"] = (1 + 0.1 * torch.randn(C, generator=g, device="cuda")).to(t)
        if case["train"]:
            state["dy"], state["dh"] = rand(rows, C), rand(rows, C)
            for n in ("x", "residual", "weight"):
                state[n].requires_grad_()
    return state


def _allowed(state, case):
    """[B,Lk] truth values, or None where every key may be attended."""
    if state["lengths"] is not None:
        return torch.arange(case["Lk"], device="cuda").view(1, -1) < state["lengths"].view(-1, 1)
    return state["mask"]


def _plain_attention(state, case):
    B, Lq, Lk, Hq, Hkv, D = (case[n] for n in ("B", "Lq", "Lk", "Hq", "Hkv", "D"))
    t, scale = state["q"].dtype, 1.0 / math.sqrt(D)
    # heads that share keys side by side: [B, Hkv, group * Lq, D]
    fold = lambda x: x.float().view(B, Lq, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)  # noqa: E731
    back = lambda x: x.view(B, Hkv, Hq // Hkv, Lq, D).permute(0, 3, 1, 2, 4).reshape(B, Lq, Hq, D).to(t)  # noqa: E731
    q, k, v = fold(state["q"]), state["k"].float().transpose(1, 2), state["v"].float().transpose(1, 2)
    ok = _allowed(state, case)
    p = torch.matmul(q, k.transpose(2, 3)).mul_(scale)
    if ok is not None:
        p.masked_fill_(~ok.view(B, 1, 1, Lk), -math.inf)
    p.sub_(p.amax(dim=-1, keepdim=True).clamp_min(-1e30)).exp_()
    p.div_(p.sum(dim=-1, keepdim=True).clamp_min(1e-30))
    out = back(torch.matmul(p, v))
    if not case["train"]:
        return out
    do = fold(state["dout"])
    dv = torch.matmul(p.transpose(2, 3), do)
    ds = torch.matmul(do, v.transpose(2, 3))
    ds.sub_((ds * p).sum(dim=-1, keepdim=True)).mul_(p).mul_(scale)
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(2, 3), q)
    return out, back(dq), dk.transpose(1, 2).to(t), dv.transpose(1, 2).to(t)


def _plain_rotary(state, case):
    x, pos, sections = state["x"], state["positions"], _sections(case)
    t = x.dtype
    axis = torch.tensor([a for a, s in enumerate(sections) for _ in range(s)], device="cuda")
    share = torch.tensor([j / s for s in sections for j in range(s)], device="cuda", dtype=torch.float64)
    angle = pos[..., axis].double() * torch.pow(10000.0, -share)
    if pos.dim() == 2:
        angle = angle.unsqueeze(0)
    c, s = angle.cos().float().unsqueeze(2), angle.sin().float().unsqueeze(2)

    def turn(z, s):
        z = z.float()
        if case["interleaved"]:
            a, b = z[..., 0::2], z[..., 1::2]
            return torch.stack([a * c - b * s, a * s + b * c], dim=-1).flatten(-2).to(t)
        a, b = z.chunk(2, dim=-1)
        return torch.cat([a * c - b * s, a * s + b * c], dim=-1).to(t)

    out = turn(x, s)
    return (out, turn(state["dout"], -s)) if case["train"] else out


def _plain_norm(state, case):
    t = state["x"].dtype
    h = state["x"].float() + state["residual"].float()
    w = state["weight"].float()
    rstd = torch.rsqrt((h * h).mean(dim=-1, keepdim=True) + 1e-6)
    n = h * rstd
    y = n * w
    if case["quantize"]:
        top = y.abs().amax(dim=-1, keepdim=True)
        scale = torch.where(top > 0, top / _E4M3_MAX, torch.ones_like(top))
        return (y / scale).to(torch.float8_e4m3fn), scale.squeeze(-1), h.to(t)
    if not case["train"]:
        return y.to(t), h.to(t)
    dy, dh = state["dy"].float(), state["dh"].float()
    dn = dy * w
    dx = dh + rstd * (dn - n * (dn * n).mean(dim=-1, keepdim=True))
    dw = (dy * n).double().sum(dim=0)
    return y.to(t), h.to(t), dx.to(t), dx.to(t), dw.to(t)


def run(state):
    case = state["case"]
    if own:
        return _own(state, case)
    plain = {"cross_attention": _plain_attention, "rotary_axes": _plain_rotary, "add_rms_norm": _plain_norm}
    with torch.no_grad():
        return plain[case["op"]](state, case)


def _own(state, case):
    import flashbev_b200 as fb
    if case["op"] == "cross_attention":
        out = fb.cross_attention(state["q"], state["k"], state["v"], key_lengths=state["lengths"], key_mask=state["mask"])
        if not case["train"]:
            return out
        return (out.detach(), *torch.autograd.grad(out, (state["q"], state["k"], state["v"]), state["dout"]))
    if case["op"] == "rotary_axes":
        out = fb.rotary_axes(state["x"], state["positions"], _sections(case), base=10000.0, interleaved=case["interleaved"])
        if not case["train"]:
            return out
        return out.detach(), torch.autograd.grad(out, state["x"], state["dout"])[0]
    if case["quantize"]:
        return fb.add_rms_norm(state["x"], state["residual"], state["weight"], eps=1e-6, quantize=True)
    y, h = fb.add_rms_norm(state["x"], state["residual"], state["weight"], eps=1e-6)
    if not case["train"]:
        return y, h
    grads = torch.autograd.grad((y, h), (state["x"], state["residual"], state["weight"]), (state["dy"], state["dh"]))
    return (y.detach(), h.detach(), *grads)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "cross_attention":
        B, Lq, Lk, Hq, Hkv, D = (case[n] for n in ("B", "Lq", "Lk", "Hq", "Hkv", "D"))
        keys = Lk * {"none": 1.0, "lengths": 0.75, "camera": 5.0 / 6.0}[case["mask"]]  # valid ones, on average
        qo, kv = B * Lq * Hq * D * size, B * keys * Hkv * D * size
        products = 2.0 * B * Hq * Lq * keys * D
        if case["train"]:
            # q, k, v, dout in, out, dq, dk, dv out; two products forward and five backward
            return {"bytes": 4 * qo + 4 * kv, "flops": 7 * products}
        return {"bytes": 2 * qo + 2 * kv, "flops": 2 * products}
    if case["op"] == "rotary_axes":
        n = case["B"] * case["L"] * case["H"] * case["D"]
        passes = 2 if case["train"] else 1
        pos = case["L"] * case["axes"] * 4 * (case["B"] if case["B"] > 1 else 1)
        return {"bytes": passes * (2 * n * size) + pos, "flops": passes * 3 * n}
    n, rows, C = case["rows"] * case["C"], case["rows"], case["C"]
    if case["quantize"]:
        return {"bytes": 3 * n * size + n + 4 * rows + C * size, "flops": 8 * n}
    if case["train"]:
        # x, residual in, y, h out; dy, dh in, dx out (one tensor serves both addends)
        return {"bytes": 7 * n * size + 2 * C * size, "flops": 18 * n}
    return {"bytes": 4 * n * size + C * size, "flops": 5 * n}


def exact(case, seed):
    """The operators' definitions in 64 bits, sample by sample and head by head."""
    state = prepare(case, seed)
    if case["op"] == "cross_attention":
        B, Lq, Lk, Hq, Hkv, D = (case[n] for n in ("B", "Lq", "Lk", "Hq", "Hkv", "D"))
        if B * Hq * Lq * Lk * D * (7 if case["train"] else 2) > 4e11:
            return None
        q, k, v = (state[n].detach().double() for n in ("q", "k", "v"))
        ok = _allowed(state, case)
        out, group = torch.zeros_like(q), Hq // Hkv
        if case["train"]:
            do = state["dout"].double()
            dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
        for b in range(B):
            seen = torch.arange(Lk, device="cuda") if ok is None else ok[b].nonzero().squeeze(-1)
            if seen.numel() == 0:
                continue
            for h in range(Hq):
                kk, vv = k[b, seen, h // group], v[b, seen, h // group]
                weights = torch.softmax(q[b, :, h] @ kk.T / math.sqrt(D), dim=-1)
                out[b, :, h] = weights @ vv
                if case["train"]:
                    g = do[b, :, h]
                    dv[b].index_put_((seen, torch.tensor(h // group, device="cuda")), weights.T @ g, accumulate=True)
                    through = weights * (g @ vv.T - (g * out[b, :, h]).sum(-1, keepdim=True)) / math.sqrt(D)
                    dq[b, :, h] = through @ kk
                    dk[b].index_put_((seen, torch.tensor(h // group, device="cuda")), through.T @ q[b, :, h], accumulate=True)
        return (out, dq, dk, dv) if case["train"] else out
    if case["op"] == "rotary_axes":
        x, sections = state["x"].detach().double(), _sections(case)
        pos = state["positions"].double().expand(case["B"], case["L"], case["axes"])
        half = case["D"] // 2
        place = (lambda p: (2 * p, 2 * p + 1)) if case["interleaved"] else (lambda p: (p, half + p))

        def turned(z, sign):
            z, y, p = z.double(), torch.zeros_like(x), 0
            for a, s in enumerate(sections):
                for j in range(s):
                    w = torch.polar(torch.ones_like(pos[..., a]), sign * pos[..., a] * 10000.0 ** (-j / s)).unsqueeze(-1)
                    i0, i1 = place(p)
                    r = torch.complex(z[..., i0], z[..., i1]) * w
                    y[..., i0], y[..., i1] = r.real, r.imag
                    p += 1
            return y

        return (turned(x, 1.0), turned(state["dout"], -1.0)) if case["train"] else turned(x, 1.0)
    x, w = (state["x"].detach().double() + state["residual"].detach().double()), state["weight"].detach().double()
    root = (x.square().sum(-1, keepdim=True) / case["C"] + 1e-6).sqrt()
    y = x / root * w
    if case["quantize"]:
        top = y.abs().amax(-1)
        return None, torch.where(top > 0, top / _E4M3_MAX, torch.ones_like(top)), x
    if not case["train"]:
        return y, x
    dy, dh = state["dy"].double(), state["dh"].double()
    inner = (dy * w * x).sum(-1, keepdim=True) / case["C"]
    dx = dh + dy * w / root - x * inner / root.pow(3)
    return y, x, dx, dx, (dy * x / root).sum(0)
