"""Operators for a view transform in which BEV queries attend to camera tokens, on libfbev.so (include/fbev_query.h).

``flash_bevpool`` lifts camera features to the BEV grid by sampling them; the operators here are what the other kind of
view transform is made of, in which every BEV cell is a query and every feature-map position a token:

  * ``cross_attention``  softmax attention of queries over keys and values of another length, with a number of valid
                         keys for each sample and / or a mask over them, key heads shared by groups of query heads;
  * ``rotary_axes``      rotary positions with several axes: (frame, row, column) of a token, (y, x) of a BEV cell;
  * ``add_rms_norm``     the residual's addition and the root-mean-square norm of the sum, optionally with an output in
                         8 bits and a scale for each row.

All of them take float32, bfloat16 and float16, compute in float32, launch on the caller's current stream and are
differentiable (once, in reverse mode).  There is no CPU path.  ``torch.jit.trace`` is refused.  The reference
(yokosyun/FlashBEV) has no counterpart.
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import Optional, Sequence

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .flash_bevpool import _DTYPES, refuse_tangents, status_pointer

_POS_DTYPES = {torch.float32: _lib.POS_F32, torch.int32: _lib.POS_I32, torch.int64: _lib.POS_I64}


def _refuse_tracing() -> None:
    """A recorded call would keep this one's result, or run with its sizes on other inputs."""
    raise RuntimeError("the query operators cannot be recorded by torch.jit.trace")


def _check_tensor(name: str, t: torch.Tensor, like: Optional[torch.Tensor] = None) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor (there is no CPU path)")
    if t.dtype not in _DTYPES:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    if like is not None and (t.dtype != like.dtype or t.device != like.device):
        raise ValueError(f"{name} must have the dtype and device of the first argument ({like.dtype}, {like.device}); "
                         f"got {t.dtype}, {t.device}")


_stream = torch._C._cuda_getCurrentRawStream  # of a device index; the handle without a Stream object around it


class _on:
    """Makes a device index current for the launch; costs nothing to speak of when it is already."""

    __slots__ = ("guard",)

    def __init__(self, index: int):
        self.guard = None if index == torch._C._cuda_getDevice() else torch.cuda.device(index)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


# What a call needs that follows from sizes, strides and types alone (checks passed, the filled C struct without its
# addresses, workspace sizes) is worked out once per such signature.  At most this many are kept of each operator.
_MOST_PLANS = 512


def _remember(plans: dict, key, plan):
    if len(plans) >= _MOST_PLANS:
        plans.clear()
    plans[key] = plan
    return plan


def _taken(t: torch.Tensor, shared_batch: bool = False) -> bool:
    """Whether the kernels take the strides of ``t`` [B,L,H,D] as they are.  A head's elements have to lie side by side.
    16-bit heads of whole 16 bytes are fetched by the copy engine, which wants strides of whole 16 bytes and no repeated
    elements, but for a whole ``shared_batch``; everything else is read element by element, whatever the strides."""
    st, size = t.stride(), t.shape
    if st[3] != 1 and size[3] != 1:
        return False
    if t.element_size() != 2 or size[3] % 8:
        return True
    return all(st[i] % 8 == 0 and (st[i] > 0 or (i == 0 and shared_batch)) for i in range(3) if size[i] > 1)


def _operand(t: torch.Tensor, shared_batch: bool = False) -> torch.Tensor:
    """``t`` itself when the kernels take it, else a contiguous copy."""
    aligned = t.data_ptr() % 16 == 0 or t.element_size() != 2 or t.shape[3] % 8 != 0
    return t if aligned and _taken(t, shared_batch) else t.clone(memory_format=torch.contiguous_format)


class _AttentionPlan:
    __slots__ = ("template", "workspace", "lse_count", "index", "direct")


_attention_plans: dict = {}


def _attention_plan(q, k, v, lengths, mask, scale) -> _AttentionPlan:
    key = (q.shape, k.shape, v.shape, q.stride(), k.stride(), v.stride(), q.dtype, k.dtype, v.dtype, q.device, k.device,
           v.device, lengths is None, None if mask is None else mask.stride(0), scale)
    plan = _attention_plans.get(key)
    if plan is not None:
        return plan
    _check_attention(q, k, v)
    plan = _AttentionPlan()
    plan.direct = _taken(q, shared_batch=True) and _taken(k) and _taken(v)
    plan.index = q.device.index
    if plan.direct:
        p = _lib.FbevAttention()
        p.struct_size = ctypes.sizeof(_lib.FbevAttention)
        p.dtype = _DTYPES[q.dtype]
        p.B, p.Lq, p.Hq, p.D = q.shape
        p.Lk, p.Hkv = k.shape[1], k.shape[2]
        p.scale = 1.0 / math.sqrt(p.D) if scale is None else scale
        p.q_shared = 1 if p.B > 1 and q.stride(0) == 0 else 0
        p.q_stride[:] = q.stride()[:3]
        p.k_stride[:] = k.stride()[:3]
        p.v_stride[:] = v.stride()[:3]
        p.mask_stride = 0 if mask is None or p.B == 1 else mask.stride(0)
        p.status = status_pointer(q.device)
        # the sizes follow from aligned addresses, which every call sees to, and from whether there are lengths
        p.q = p.k = p.v = 4096
        p.key_lengths = None if lengths is None else 4096
        lib = _lib.load()
        plan.workspace = tuple(lib.fbev_cross_attention_workspace_bytes(ctypes.byref(p), i) for i in (0, 1))
        plan.lse_count = lib.fbev_cross_attention_lse_count(ctypes.byref(p))
        p.q = p.k = p.v = p.key_lengths = None
        plan.template = bytes(p)
    return _remember(_attention_plans, key, plan)


def _planned(q, k, v, lengths, mask, scale):
    """The plan of a call and its operands, copied where the kernels do not take them as they are."""
    plan = _attention_plan(q, k, v, lengths, mask, scale)
    if not plan.direct or (q.data_ptr() | k.data_ptr() | v.data_ptr()) & 15:
        q, k, v = _operand(q, shared_batch=True), _operand(k), _operand(v)
        plan = _attention_plan(q, k, v, lengths, mask, scale)
    return plan, q, k, v


def _attention_problem(plan, q, k, v, lengths, mask, backward):
    """The filled struct and the workspace, which has to live until the launch is queued."""
    p = _lib.FbevAttention.from_buffer_copy(plan.template)
    p.q, p.k, p.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    if not p.status:  # a plan made while a graph was captured
        p.status = status_pointer(q.device)
    if lengths is not None:
        p.key_lengths = lengths.data_ptr()
    if mask is not None:
        p.key_mask = mask.data_ptr()
    nbytes = plan.workspace[backward]
    if not nbytes:
        return p, None
    ws = q.new_empty(nbytes, dtype=torch.uint8)
    p.workspace, p.workspace_bytes = ws.data_ptr(), nbytes
    return p, ws


def _attention_forward(plan, q, k, v, lengths, mask, with_lse):
    with _on(plan.index):
        p, ws = _attention_problem(plan, q, k, v, lengths, mask, 0)
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        lse = q.new_empty(plan.lse_count, dtype=torch.float32) if with_lse else None
        rc = _lib.load().fbev_cross_attention(ctypes.byref(p), out.data_ptr(), None if lse is None else lse.data_ptr(),
                                              _stream(plan.index))
    if rc:
        _lib.check(rc, "fbev_cross_attention")
    return out, lse


class _CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths, mask, scale, plan):
        out, lse = _attention_forward(plan, q, k, v, lengths, mask, True)
        ctx.save_for_backward(q, k, v, lengths, mask, out, lse)
        ctx.scale = scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        q, k, v, lengths, mask, out, lse = ctx.saved_tensors
        need_q, need_kv = ctx.needs_input_grad[0], ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        gq = gk = gv = None
        # saved tensors may come back at other addresses or strides (a hook moved them)
        plan, q, k, v = _planned(q, k, v, lengths, mask, ctx.scale)
        with _on(plan.index):
            go = grad_out.contiguous()
            if go.data_ptr() % 16:
                go = go.clone()
            p, ws = _attention_problem(plan, q, k, v, lengths, mask, 1)
            if need_q:
                gq = torch.empty_like(q, memory_format=torch.contiguous_format)
            if need_kv:
                gk = torch.empty_like(k, memory_format=torch.contiguous_format)
                gv = torch.empty_like(v, memory_format=torch.contiguous_format)
            rc = _lib.load().fbev_cross_attention_grad(
                ctypes.byref(p), out.data_ptr(), lse.data_ptr(), go.data_ptr(), gq.data_ptr() if need_q else None,
                gk.data_ptr() if need_kv else None, gv.data_ptr() if need_kv else None, _stream(plan.index))
        if rc:
            _lib.check(rc, "fbev_cross_attention_grad")
        return gq, gk if ctx.needs_input_grad[1] else None, gv if ctx.needs_input_grad[2] else None, None, None, None, None


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, key_lengths: Optional[torch.Tensor] = None,
                    key_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """Softmax attention of queries over an encoder's tokens.

    Args:
        q: queries [B,Lq,Hq,D].  A batch expanded from one sample (stride 0) is read once.
        k, v: keys and values [B,Lk,Hkv,D]; Hq must be a multiple of Hkv, and query head h uses key head
            h // (Hq // Hkv).  D is 1 to 128.  Views with strides of whole 16 bytes are taken as they are (for instance
            slices of one projection's output), others are copied.
        key_lengths: [B] int32 or int64: only the first so many keys of a sample may be attended (clamped to 0..Lk).
        key_mask: [B,Lk] or [Lk] bool, True where a key may be attended.  Both may be given: both must allow.
        scale: factor of the scores; default 1 / sqrt(D).  At most 1e30 in magnitude.
    Returns:
        [B,Lq,Hq,D] in the dtype of q.  Rows that may attend nothing are zero, and so are their gradients.  What
        stands in keys and values that may not be attended (infinities, NaN) has no influence.  A row with a NaN or
        +infinity among its scores, or with none above -infinity, is NaN, as are the gradients it reaches.

    Scores, softmax statistics and sums are float32; for 16-bit inputs the softmax weights are rounded to the input's
    type before they meet the values, as are the score gradients before they meet queries and keys: in float16 those lose
    what is below 2^-24 and overflow beyond 65504, so train with a scaled loss there, as with any float16 gradient.  One
    in eight of these weights, in the gradients two in eight, comes from a cubic whose relative error, 2^-13.7, is below
    that rounding (bfloat16 2^-8, float16 2^-11).
    float32 operands, and 16-bit heads of a width that is not a multiple of eight, enter the products as three bfloat16
    parts each, which keeps 24 bits; an infinity (or a value beyond 3.38e38) among such operands that are attended gives
    NaN.  Gradients are the same from run to run.  With few
    queries the keys are split over the GPU and the parts joined.

    The kernels' waits are bounded (about two seconds): one that runs out leaves a result that is not valid and raises a
    flag, which ``device_status()`` reads.
    """
    if torch._C._is_tracing():
        _refuse_tracing()
    refuse_tangents(q, k, v)
    if scale is not None:
        scale = float(scale)
        if not abs(scale) <= _lib.ATTENTION_MAX_SCALE:
            raise ValueError(f"scale must be finite and at most {_lib.ATTENTION_MAX_SCALE:g} in magnitude, got {scale}")
    if key_lengths is not None or key_mask is not None:
        if k.dim() != 4:
            _check_attention(q, k, v)
        key_lengths, key_mask = _attention_masks(q, k, key_lengths, key_mask)
    plan, q, k, v = _planned(q, k, v, key_lengths, key_mask, scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _CrossAttention.apply(q, k, v, key_lengths, key_mask, scale, plan)
    return _attention_forward(plan, q, k, v, key_lengths, key_mask, False)[0]


def _check_attention(q, k, v) -> None:
    _check_tensor("q", q)
    _check_tensor("k", k, q)
    _check_tensor("v", v, q)
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise ValueError(f"q must be [B,Lq,Hq,D] and k, v [B,Lk,Hkv,D]; got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if not 1 <= q.shape[3] <= 128:
        raise ValueError(f"the head width must be 1 to 128, got {q.shape[3]}")
    if k.shape[2] == 0 or q.shape[2] == 0 or q.shape[2] % k.shape[2] != 0:
        raise ValueError(f"the number of query heads ({q.shape[2]}) must be a multiple of the key heads ({k.shape[2]})")


def _attention_masks(q, k, key_lengths, key_mask):
    B, Lk = k.shape[:2]
    if key_lengths is not None:
        if key_lengths.shape != (B,) or key_lengths.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"key_lengths must be int32 or int64 of shape [{B}]")
        if key_lengths.dtype == torch.int64:
            key_lengths = key_lengths.clamp(0, Lk)
        if key_lengths.dtype != torch.int32 or key_lengths.device != q.device or not key_lengths.is_contiguous():
            key_lengths = key_lengths.to(device=q.device, dtype=torch.int32).contiguous()
    if key_mask is not None:
        if key_mask.dtype != torch.bool or key_mask.shape not in ((B, Lk), (Lk,)):
            raise ValueError(f"key_mask must be bool of shape [{B},{Lk}] or [{Lk}]")
        if key_mask.device != q.device:
            key_mask = key_mask.to(q.device)
        if key_mask.dim() == 1:
            key_mask = key_mask.unsqueeze(0).expand(B, Lk)
        if Lk > 1 and key_mask.stride(1) != 1:
            key_mask = key_mask.contiguous()
    return key_lengths, key_mask


@functools.lru_cache(maxsize=64)
def _rotary_table(sections, base):
    """(turns per unit of position, axis) of every pair: 2 pi * turns = base ** (-j / S) for pair j of an axis with S."""
    turns, axis = (ctypes.c_double * _lib.ROTARY_MAX_PAIRS)(), (ctypes.c_uint8 * _lib.ROTARY_MAX_PAIRS)()
    i = 0
    for a, s in enumerate(sections):
        for j in range(s):
            turns[i], axis[i] = base ** (-j / s) / (2.0 * math.pi), a
            i += 1
    return turns, axis


_rotary_plans: dict = {}


def _rotary(x, positions, sections, base, interleaved, inverse):
    key = (x.shape, x.stride(), x.dtype, positions.dtype, positions.dim(), sections, base, interleaved, inverse)
    template = _rotary_plans.get(key)
    if template is None:
        p = _lib.FbevRotary()
        p.struct_size = ctypes.sizeof(_lib.FbevRotary)
        p.dtype = _DTYPES[x.dtype]
        p.B, p.L, p.H, p.D = x.shape
        p.pairs, p.axes = sum(sections), len(sections)
        p.interleaved, p.inverse = int(interleaved), int(inverse)
        p.pos_dtype = _POS_DTYPES[positions.dtype]
        p.x_stride[:] = x.stride()[:3]
        p.pos_stride = 0 if positions.dim() == 2 else positions.stride(0)
        p.pair_turns, p.pair_axis = _rotary_table(sections, base)
        template = _remember(_rotary_plans, key, bytes(p))
    p = _lib.FbevRotary.from_buffer_copy(template)
    p.x, p.positions = x.data_ptr(), positions.data_ptr()
    index = x.device.index
    out = torch.empty_like(x, memory_format=torch.contiguous_format)
    with _on(index):
        rc = _lib.load().fbev_rotary_axes(ctypes.byref(p), out.data_ptr(), _stream(index))
    if rc:
        _lib.check(rc, "fbev_rotary_axes")
    return out


def _rotary_operand(x, interleaved):
    """x with a head's elements side by side, and in the interleaved layout with whole pairs addressable at once."""
    good = x.stride(3) == 1 or x.shape[3] == 1
    if interleaved:
        good = good and x.data_ptr() % (2 * x.element_size()) == 0
        good = good and all(s % 2 == 0 for s, n in zip(x.stride()[:3], x.shape) if n > 1)
    return x if good else x.clone(memory_format=torch.contiguous_format)


class _RotaryAxes(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, sections, base, interleaved):
        ctx.save_for_backward(positions)
        ctx.args = (sections, base, interleaved)
        return _rotary(x, positions, sections, base, interleaved, False)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        positions, = ctx.saved_tensors
        sections, base, interleaved = ctx.args
        return _rotary(_rotary_operand(grad, interleaved), positions, sections, base, interleaved, True), None, None, None, None


def rotary_axes(x: torch.Tensor, positions: torch.Tensor, sections: Sequence[int], *, base: float = 10000.0,
                interleaved: bool = False) -> torch.Tensor:
    """Rotary positions with several axes.

    Args:
        x: [B,L,H,D], D up to 256, strided views allowed.
        positions: [L,A] or [B,L,A], float32, int32 or int64: the coordinates of every token on A axes (1 to 8).
        sections: A numbers: how many pairs of elements turn with each axis.  The first ``2 * sum(sections)`` elements
            of a head are rotated, the rest is copied.
        base: pair j of an axis with S pairs turns by ``position * base ** (-j / S)``.
        interleaved: pairs are neighbours (2p, 2p + 1); otherwise (p, P + p) with P = sum(sections).
    Returns:
        A new tensor like x (contiguous).  The gradient with respect to x is the opposite rotation; positions carry none.

    Angles are formed and reduced in float64: frequency and product round there, with the default base by at most
    |angle| * 2^-49 together, which float32 does not show up to angles of 2^24 radians.
    """
    if torch._C._is_tracing():
        _refuse_tracing()
    refuse_tangents(x, positions)
    sections, base, interleaved = tuple(sections), float(base), bool(interleaved)
    if not all(isinstance(s, int) for s in sections):  # the key below does not tell 4.0 from 4
        raise ValueError(f"sections must be whole numbers, got {sections}")
    key = (x.shape, x.dtype, x.device, positions.shape, positions.dtype, positions.device, sections, base, interleaved)
    if key not in _rotary_checked:
        _check_rotary(x, positions, sections, base, interleaved)
        _remember(_rotary_checked, key, True)
    if positions.requires_grad:
        raise ValueError("positions carry no gradient; detach them")
    positions = positions.contiguous()
    x = _rotary_operand(x, interleaved)
    if torch.is_grad_enabled() and x.requires_grad:
        return _RotaryAxes.apply(x, positions, sections, base, interleaved)
    return _rotary(x, positions, sections, base, interleaved, False)


_rotary_checked: dict = {}


def _check_rotary(x, positions, sections, base, interleaved) -> None:
    _check_tensor("x", x)
    if x.dim() != 4 or not 1 <= x.shape[3] <= 256:
        raise ValueError(f"x must be [B,L,H,D] with D from 1 to 256, got {tuple(x.shape)}")
    if not 1 <= len(sections) <= 8 or min(sections) < 0 or 2 * sum(sections) > x.shape[3]:
        raise ValueError(f"sections must be 1 to 8 non-negative whole numbers with 2 * sum <= {x.shape[3]}, got {sections}")
    B, L = x.shape[:2]
    if positions.shape not in ((L, len(sections)), (B, L, len(sections))):
        raise ValueError(f"positions must be [{L},{len(sections)}] or [{B},{L},{len(sections)}], got {tuple(positions.shape)}")
    if positions.dtype not in _POS_DTYPES:
        raise ValueError(f"positions must be float32, int32 or int64, got {positions.dtype}")
    if positions.device != x.device:
        raise ValueError("positions are on another device than x")
    if not (math.isfinite(base) and base > 0):
        raise ValueError("base must be positive and finite")
    if interleaved and x.shape[3] % 2:
        raise ValueError("interleaved pairs need an even D")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _norm_forward(x, residual, weight, eps, with_rstd):
    C = x.shape[-1]
    rows = x.numel() // C
    index = x.device.index
    y = torch.empty_like(x)
    h = torch.empty_like(x) if residual is not None else None
    rstd = x.new_empty(rows, dtype=torch.float32) if with_rstd else None
    with _on(index):
        rc = _lib.load().fbev_add_rms_norm(_DTYPES[x.dtype], rows, C, eps, x.data_ptr(), _ptr(residual), _ptr(weight),
                                           y.data_ptr(), _ptr(h), _ptr(rstd), _stream(index))
    if rc:
        _lib.check(rc, "fbev_add_rms_norm")
    return y, h, rstd


class _AddRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        y, h, rstd = _norm_forward(x, residual, weight, eps, True)
        ctx.save_for_backward(x if h is None else h, weight, rstd)
        ctx.set_materialize_grads(False)
        return y if h is None else (y, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y, grad_h=None):
        h, weight, rstd = ctx.saved_tensors
        if grad_y is None:  # only the sum was used
            return grad_h, grad_h if ctx.needs_input_grad[1] else None, None, None
        lib = _lib.load()
        C = h.shape[-1]
        rows = h.numel() // C
        dev = h.device
        need_x = ctx.needs_input_grad[0] or ctx.needs_input_grad[1]
        need_w = ctx.needs_input_grad[2]
        with _on(dev.index):
            grad_y = grad_y.contiguous()
            grad_h = None if grad_h is None else grad_h.contiguous()
            gx = torch.empty_like(h) if need_x else None
            gw = torch.empty_like(weight) if need_w else None
            nbytes = lib.fbev_add_rms_norm_grad_workspace_bytes(rows, C, int(need_w))
            ws = h.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
            rc = lib.fbev_add_rms_norm_grad(_DTYPES[h.dtype], rows, C, h.data_ptr(), rstd.data_ptr(), _ptr(weight),
                                            grad_y.data_ptr(), _ptr(grad_h), _ptr(gx), _ptr(gw), _ptr(ws), nbytes,
                                            _stream(dev.index))
        if rc:
            _lib.check(rc, "fbev_add_rms_norm_grad")
        return (gx if ctx.needs_input_grad[0] else None, gx if ctx.needs_input_grad[1] else None, gw, None)


def add_rms_norm(x: torch.Tensor, residual: Optional[torch.Tensor] = None, weight: Optional[torch.Tensor] = None, *,
                 eps: float = 1e-6, quantize: bool = False):
    """Residual addition and root-mean-square norm over the last dimension.

    ``h = x + residual``, ``y = h / sqrt(mean(h ** 2) + eps) * weight``, in float32 from the unrounded sum (the squares of a
    row have to stay within float32).

    Args:
        x: [..., C].  residual: the same shape, or None.  weight: [C], or None for ones.  All of one dtype.
        quantize: y in 8 bits for a matrix product in float8: every row is divided by a scale of its own, max|y| / 448
            (1 for a row of zeros), and rounded to float8_e4m3fn.  Serving only: no gradient.
    Returns:
        (y, h), or (q, scales, h) with ``quantize``: q like y in float8_e4m3fn, scales [...] float32, y ~ q * scales.
        Without a residual h is x itself.

    The gradient reads h as it was returned, rounded to its type, and the root as the forward formed it.
    """
    if torch._C._is_tracing():
        _refuse_tracing()
    refuse_tangents(x, residual, weight)
    key = (x.shape, x.dtype, x.device, None if residual is None else (residual.shape, residual.dtype, residual.device),
           None if weight is None else (weight.shape, weight.dtype, weight.device))
    if key not in _norm_checked:
        _check_norm(x, residual, weight)
        _remember(_norm_checked, key, True)
    if not 0.0 <= eps < math.inf:
        raise ValueError("eps must be finite and not negative")
    given, x = x, x.contiguous()
    residual = None if residual is None else residual.contiguous()
    weight = None if weight is None else weight.contiguous()
    grad = torch.is_grad_enabled() and (
        x.requires_grad or (residual is not None and residual.requires_grad) or (weight is not None and weight.requires_grad))
    if quantize:
        if grad:
            raise ValueError("the 8-bit output carries no gradient; call under torch.no_grad()")
        lib = _lib.load()
        C = x.shape[-1]
        dev = x.device
        q = torch.empty_like(x, dtype=torch.float8_e4m3fn)
        scales = x.new_empty(x.shape[:-1], dtype=torch.float32)
        h = torch.empty_like(x) if residual is not None else None
        with _on(dev.index):
            rc = lib.fbev_add_rms_norm_e4m3(_DTYPES[x.dtype], x.numel() // C, C, eps, x.data_ptr(), _ptr(residual), _ptr(weight),
                                            q.data_ptr(), scales.data_ptr(), _ptr(h), _stream(dev.index))
        if rc:
            _lib.check(rc, "fbev_add_rms_norm_e4m3")
        return q, scales, given if h is None else h
    if not grad:
        y, h, _ = _norm_forward(x, residual, weight, eps, False)
        return y, given if h is None else h
    if residual is None:
        return _AddRmsNorm.apply(x, None, weight, eps), given
    return _AddRmsNorm.apply(x, residual, weight, eps)


_norm_checked: dict = {}


def _check_norm(x, residual, weight) -> None:
    _check_tensor("x", x)
    if x.dim() < 1 or not 1 <= x.shape[-1] <= 1 << 20:
        raise ValueError(f"x must be [..., C] with C from 1 to 2^20, got {tuple(x.shape)}")
    if residual is not None:
        _check_tensor("residual", residual, x)
        if residual.shape != x.shape:
            raise ValueError(f"residual must have the shape of x {tuple(x.shape)}, got {tuple(residual.shape)}")
    if weight is not None:
        _check_tensor("weight", weight, x)
        if weight.shape != x.shape[-1:]:
            raise ValueError(f"weight must have shape [{x.shape[-1]}], got {tuple(weight.shape)}")
