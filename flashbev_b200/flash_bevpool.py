"""``FlashBEVPool`` / ``flash_bevpool``: the operator of the reference package, on libfbev.so.

Mirrors flashbev/flashbevpool/flash_bevpool.py of the reference:
  * ``FlashBEVPool.forward`` keeps the 14 positional slots of flash_bevpool.py:22-23 and
    ``backward`` returns the 14-tuple of :135-136 (gradients for depth and features only);
  * ``flash_bevpool`` keeps names, order and defaults of :139-140 and reorders its first
    two arguments exactly as :163-166 does.

Differences, all additive or host-side:
  * no host synchronisation per call: sizes come from a cached host copy of ``grid_size``;
    ``roi_range``, ``image_size`` and ``feature_size`` are read on the device, as the
    reference's backward kernel already does (flash_bevpool_cuda.cu:465-470);
  * launches go to the caller's current stream (the reference uses the legacy default
    stream, flash_bevpool_cuda.cu:807);
  * float32, bfloat16 and float16 features are processed natively (float32 accumulation)
    and the output has the feature dtype; the reference up-casts to float32 (:47-49);
  * ``depth_distribution=2`` selects the categorical depth mode (depth = probabilities
    [B,N,H,W,D]); ``pool``, ``depth_bin_range``, ``legacy_depth_grad``, ``deterministic`` and
    ``y_range`` are keyword-only extras of the wrapper;
  * the kernel-variant flags (``use_shared_memory``, ``optimize_z_precompute``,
    ``use_warp_kernel``, ``use_vectorized_load``) are accepted and ignored: they select
    between reference kernels that compute the same thing;
  * ``projection_matrices`` may be [B,N,3,4] or [B,N,4,4] (rows 0-2 are used).

There is no CPU path: tensors must live on a CUDA device and libfbev.so must load.
"""
from __future__ import annotations

import ctypes
import enum
import weakref
from typing import Optional, Tuple

import numpy as np
import torch
from torch.autograd import forward_ad

from . import _lib

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def refuse_tangents(*tensors) -> None:
    """Calls without gradients do not go through the autograd functions, which would refuse forward-mode differentiation:
    the tangents would be lost without a word."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("forward-mode differentiation is not supported")


class DepthSpec(int):
    """``depth_distribution`` with the extra options riding along.

    It is an ``int`` (0 gaussian, 1 laplace, 2 categorical probabilities, 3 categorical logits: the softmax over
    the bins is folded into the operator), so it fits the reference's positional slot; the attributes carry what
    the reference has no slot for.
    """

    def __new__(cls, mode: int, pool: Optional[str] = None, depth_bin_range: Optional[Tuple[float, float]] = None,
                legacy_depth_grad: bool = False, y_range: Optional[Tuple[int, int]] = None,
                out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None, host_row_chunks: int = 0,
                save_lists: bool = False, compact_rows: bool = False, deterministic: bool = False):
        mode = int(mode)
        if mode not in (0, 1, 2, 3):
            raise ValueError("depth_distribution must be 0 (gaussian), 1 (laplace), 2 (categorical probabilities) or "
                             f"3 (categorical logits), got {mode}")
        self = super().__new__(cls, mode)
        if pool is None:
            pool = "sum" if mode >= 2 else "mean"
        if pool not in ("mean", "sum"):
            raise ValueError(f"pool must be 'mean' or 'sum', got {pool!r}")
        self.pool = pool
        if mode >= 2:
            if depth_bin_range is None:
                raise ValueError("depth_distribution=2 / 3 needs depth_bin_range=(first_edge, bin_width)")
            d0, delta = float(depth_bin_range[0]), float(depth_bin_range[1])
            if not delta > 0:
                raise ValueError("depth_bin_range: bin width must be positive")
        else:
            d0, delta = 0.0, 1.0
        self.d0, self.delta = d0, delta
        self.legacy_depth_grad = bool(legacy_depth_grad)
        self.deterministic = bool(deterministic)
        self.y_range = None if y_range is None else (int(y_range[0]), int(y_range[1]))
        if out_dtype not in (None, torch.float32):
            raise ValueError("out_dtype must be None (the feature dtype) or torch.float32")
        self.out_dtype = out_dtype
        self.out = out
        self.save_lists = bool(save_lists)
        self.compact_rows = bool(compact_rows)
        if self.compact_rows and y_range is None:
            raise ValueError("compact_rows needs y_range")
        self.host_row_chunks = int(host_row_chunks)
        if not 0 <= self.host_row_chunks <= 16:
            raise ValueError("host_row_chunks must be 0 (the kernel stores to the host buffer) or 1..16 row bands")
        return self


# host copies of small device tensors, keyed by the identity of the tensor object; the weak
# reference drops the entry when the tensor dies, the version catches in-place changes
_host_cache = {}


def _host_values(t: torch.Tensor) -> tuple:
    """Values of a small tensor on the host.  Synchronises only the first time a given
    (tensor, version) is seen; the reference synchronises on every call (flash_bevpool.py:58-67).
    A caller that builds a new device ``grid_size`` tensor for every call (as the reference's
    tools/utils/data_utils.py:208-209 does once per benchmark) pays that one synchronisation per
    call and leaves no entry behind (the weak reference removes it with the tensor); keeping the
    tensor, or passing a host tensor, avoids it."""
    if t.device.type == "cpu":
        return tuple(t.tolist())
    key = id(t)
    hit = _host_cache.get(key)
    if hit is not None and hit[0]() is t and hit[1] == t._version:
        return hit[2]
    vals = tuple(t.tolist())
    _host_cache[key] = (weakref.ref(t, lambda _r, k=key: _host_cache.pop(k, None)), t._version, vals)
    return vals


_status_words = {}


def status_word(device: torch.device) -> torch.Tensor:
    """Per-device int32 word the kernels OR FBEV_DEV_* flags into (never read on the hot path)."""
    key = (device.type, device.index if device.index is not None else torch.cuda.current_device())
    w = _status_words.get(key)
    if w is None:
        with torch.inference_mode(False):
            w = torch.zeros(1, dtype=torch.int32, device=device)
        # kernels on any stream may write to it from now on; a thread that made one at the same time keeps this one
        torch.cuda.current_stream(device).synchronize()
        w = _status_words.setdefault(key, w)
    return w


def status_pointer(device: torch.device) -> Optional[int]:
    """Address of the device's status word for a call.  None while a graph is captured before any other call has made the
    word: made there, its memory would be the graph's and every replay would clear it."""
    key = (device.type, device.index if device.index is not None else torch.cuda.current_device())
    if key not in _status_words:
        with torch.cuda.device(device):
            if torch.cuda.is_current_stream_capturing():
                return None
    return status_word(device).data_ptr()


class DeviceStatus(enum.IntFlag):
    """What kernels found wrong while they ran (FBEV_DEV_* of include/fbev.h and include/fbev_query.h)."""
    OK = 0
    BAD_FEATURE_SIZE = _lib.DEV_BAD_FEATURE_SIZE  # a feature_size larger than the tensor; that camera was skipped
    TIMEOUT = _lib.DEV_TIMEOUT                    # a wait inside an attention kernel ran out; its output is not valid


def device_status(device=None, *, clear: bool = False) -> DeviceStatus:
    """Flags that the operators' kernels raised on a CUDA device (default: the current one) since they were last cleared.

    Calls do not read them: a kernel has no other way to tell, and reading would make every call wait.  This function
    waits for all work on the device, so call it where a program synchronises anyway (after a step, before results are
    used).  ``clear`` forgets the flags that are returned.  A graph captured before the device's first call outside a
    capture reports nothing.
    """
    device = torch.device("cuda" if device is None else device)
    if device.type != "cuda":
        raise ValueError(f"device must be a CUDA device, got {device}")
    index = torch.cuda.current_device() if device.index is None else device.index
    with torch.cuda.device(index):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("device_status waits for the device; call it outside graph capture")
        w = _status_words.get(("cuda", index))
        if w is None:  # no call yet
            return DeviceStatus.OK
        torch.cuda.synchronize(index)
        flags = int(w.item())
        if clear and flags:
            w.bitwise_and_(~flags)
            torch.cuda.current_stream(index).synchronize()
    return DeviceStatus(flags)


_workspaces = {}


def workspace(device: torch.device, stream_ptr: int) -> torch.Tensor:
    """Zero-initialised scheduler words for calls on (device, stream).  Calls on one stream run in
    order and each leaves the words zero, so one buffer per stream is enough."""
    key = (device.index if device.index is not None else torch.cuda.current_device(), int(stream_ptr))
    w = _workspaces.get(key)
    if w is None:
        w = torch.zeros(_lib.WORKSPACE_BYTES // 4, dtype=torch.int32, device=device)
        _workspaces[key] = w
    return w


def _on(t: torch.Tensor, device: torch.device, dtype: torch.dtype) -> torch.Tensor:
    if t.device != device or t.dtype != dtype:
        t = t.to(device=device, dtype=dtype)
    return t if t.is_contiguous() else t.contiguous()


class _on_device:
    """Device guard that costs nothing when ``device`` is already current (the usual case; the library
    launches on the current device, so a call for another device must switch)."""

    __slots__ = ("guard",)

    def __init__(self, device: torch.device):
        idx = device.index
        self.guard = None if idx is None or idx == torch.cuda.current_device() else torch.cuda.device(device)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def make_problem(depth_params, image_feats, projection_matrices, feature_size, image_size, roi_range, grid_size,
                 spec: DepthSpec, epsilon: float, threshold: float):
    """Builds the FbevProblem for a call and returns it with the tensors that must stay alive."""
    if not image_feats.is_cuda:
        raise RuntimeError("flash_bevpool runs on CUDA tensors only (there is no CPU path)")
    dev = image_feats.device
    dtype = image_feats.dtype if image_feats.dtype in _DTYPES else torch.float32
    feats = _on(image_feats, dev, dtype)
    depth = _on(depth_params, dev, dtype)
    proj = _on(projection_matrices, dev, torch.float32)
    fsize = _on(feature_size, dev, torch.int32)
    isize = _on(image_size, dev, torch.int32)
    roi = _on(roi_range, dev, torch.float32)
    if feats.dim() != 5 or depth.dim() != 5 or feats.shape[:4] != depth.shape[:4]:
        raise ValueError(f"image_feats must be [B,N,H,W,C] and depth_params [B,N,H,W,D]; got "
                         f"{tuple(image_feats.shape)} and {tuple(depth_params.shape)}")
    B, N, H, W, C = feats.shape
    if proj.dim() != 4 or tuple(proj.shape[:2]) != (B, N) or tuple(proj.shape[2:]) not in ((3, 4), (4, 4)):
        raise ValueError(f"projection_matrices must be [B,N,3,4] or [B,N,4,4]; got {tuple(proj.shape)}")
    if fsize.numel() != B * N * 2 or isize.numel() != 2 or roi.numel() != 6:
        raise ValueError("feature_size must be [B,N,2], image_size [2], roi_range [6]")
    grid = _host_values(grid_size)
    if len(grid) != 3:
        raise ValueError("grid_size must hold [grid_x, grid_y, grid_z]")
    X, Y, Z = (int(v) for v in grid)
    p = _lib.FbevProblem()
    p.struct_size = ctypes.sizeof(_lib.FbevProblem)
    p.dtype = _DTYPES[dtype]
    p.out_dtype = _lib.F32 if spec.out_dtype == torch.float32 else p.dtype
    p.B, p.N, p.H, p.W, p.C = B, N, H, W, C
    p.D = depth.shape[-1]
    p.X, p.Y, p.Z = X, Y, Z
    p.proj_stride = proj.shape[2] * proj.shape[3]
    p.mode = int(spec)
    p.pool = _lib.POOL_SUM if spec.pool == "sum" else _lib.POOL_MEAN
    p.epsilon, p.threshold = float(epsilon), float(threshold)
    p.depth_d0, p.depth_delta = spec.d0, spec.delta
    yb, ye = spec.y_range if spec.y_range is not None else (0, Y)
    p.y_begin, p.y_end = yb, ye
    p.compact_rows = 1 if spec.compact_rows else 0
    p.image_feats, p.depth, p.projection = feats.data_ptr(), depth.data_ptr(), proj.data_ptr()
    p.feature_size, p.image_size, p.roi_range = fsize.data_ptr(), isize.data_ptr(), roi.data_ptr()
    p.status = status_pointer(dev)
    p.workspace = workspace(dev, torch.cuda.current_stream(dev).cuda_stream).data_ptr()
    keep = (feats, depth, proj, fsize, isize, roi)
    if int(spec) == _lib.DEPTH_CATEGORICAL_LOGITS:
        # scratch for the per-texel softmax statistics; every call fills it itself
        stats = torch.empty(B * N * H * W * 2, dtype=torch.float32, device=dev)
        p.depth_stats = stats.data_ptr()
        keep = keep + (stats,)
    return p, keep


def _out_dtype(spec: DepthSpec, feats: torch.Tensor) -> torch.dtype:
    return torch.float32 if spec.out_dtype == torch.float32 else feats.dtype


# host tensors already found page-locked, keyed by the identity of the tensor object (Tensor.is_pinned asks the
# driver about the address, tens of microseconds every time); the weak reference drops the entry with the tensor
_pinned_seen = {}


def _is_pinned(t: torch.Tensor) -> bool:
    key = id(t)
    hit = _pinned_seen.get(key)
    if hit is not None and hit[0]() is t and hit[1] == t.data_ptr():
        return True
    if not t.is_pinned():
        return False
    _pinned_seen[key] = (weakref.ref(t, lambda _r, k=key: _pinned_seen.pop(k, None)), t.data_ptr())
    return True


def _check_out(out, shape, dtype, device, partial, needs_grad):
    """A caller-provided result buffer: a tensor on the operator's device, or page-locked host memory that
    the kernel writes through the bus directly (the device-to-host copy of the result disappears)."""
    if tuple(out.shape) != tuple(shape) or out.dtype != dtype or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {dtype} tensor of shape {tuple(shape)}")
    if out.is_cuda:
        if out.device != device:
            raise ValueError("out is on another device than image_feats")
        if partial:
            out.zero_()
        return out
    if not _is_pinned(out):
        raise ValueError("a host out tensor must be page-locked (tensor.pin_memory())")
    if partial:
        raise ValueError("y_range with a host out tensor is not supported")
    if needs_grad:
        raise ValueError("a host out tensor cannot carry gradients; call under torch.no_grad()")
    return out


def _forward(depth_params, image_feats, projection_matrices, feature_size, image_size, roi_range, grid_size, spec,
             epsilon, depth_weight_threshold, needs_grad):
    """One forward launch; returns (out, problem, kept tensors)."""
    p, keep = make_problem(depth_params, image_feats, projection_matrices, feature_size, image_size,
                           roi_range, grid_size, spec, epsilon, depth_weight_threshold)
    feats = keep[0]
    dev = feats.device
    shape = (p.B, p.y_end - p.y_begin if spec.compact_rows else p.Y, p.X, p.C)
    partial = (p.y_begin, p.y_end) != (0, p.Y) and not spec.compact_rows
    if spec.out is not None:
        out = _check_out(spec.out, shape, _out_dtype(spec, feats), dev, partial, needs_grad)
    else:
        out = (torch.zeros if partial else torch.empty)(shape, dtype=_out_dtype(spec, feats), device=dev)
    lib = _lib.load()
    if needs_grad and spec.save_lists:
        # a backward will follow and the caller asked for it: the forward leaves it the lists it builds (FbevProblem.saved_state)
        nbytes = lib.fbev_saved_state_bytes(ctypes.byref(p))
        if nbytes:
            lists = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            p.saved_state, p.saved_state_bytes = lists.data_ptr(), nbytes
            keep = keep + (lists,)
    with _on_device(dev):
        stream = torch.cuda.current_stream(dev).cuda_stream
        if spec.out is not None and not out.is_cuda and spec.host_row_chunks > 0:
            # bands of rows: the copy engine moves one band to the host while the next is computed
            staging = torch.empty(shape, dtype=out.dtype, device=dev)
            rc = lib.fbev_forward_to_host(ctypes.byref(p), staging.data_ptr(), out.data_ptr(), spec.host_row_chunks,
                                          stream)
            _lib.check(rc, "fbev_forward_to_host")
        else:
            rc = lib.fbev_forward(ctypes.byref(p), out.data_ptr(), None, stream)
            if rc:
                _lib.check(rc, "fbev_forward")
    return out, p, keep


class FlashBEVPool(torch.autograd.Function):
    """Fused BEV pooling: projection, depth weight, bilinear sampling and the reduction over
    cameras and height bins in one kernel; see the module docstring for the contract."""

    @staticmethod
    def forward(ctx, depth_params, image_feats, projection_matrices, feature_size, image_size, roi_range,
                grid_size, depth_distribution=0, use_shared_memory=True, optimize_z_precompute=True,
                use_warp_kernel=False, use_vectorized_load=False, epsilon=1e-6, depth_weight_threshold=1e-6):
        spec = depth_distribution if isinstance(depth_distribution, DepthSpec) else DepthSpec(depth_distribution)
        out, p, keep = _forward(depth_params, image_feats, projection_matrices, feature_size, image_size, roi_range,
                                grid_size, spec, epsilon, depth_weight_threshold,
                                depth_params.requires_grad or image_feats.requires_grad)
        ctx.save_for_backward(*keep[:6])
        ctx.held = keep[6:]  # scratch of the call that the backward reads again (saved lists, softmax statistics)
        ctx.spec = spec
        ctx.problem = p  # the backward launches on the same tensors: same struct, as long as their addresses hold
        ctx.grid = (p.X, p.Y, p.Z)
        ctx.epsilon = float(epsilon)
        ctx.depth_weight_threshold = float(depth_weight_threshold)
        ctx.in_dtypes = (depth_params.dtype, image_feats.dtype)
        return out

    @staticmethod
    def backward(ctx, out_grad):
        feats, depth, proj, fsize, isize, roi = ctx.saved_tensors[:6]
        spec = ctx.spec
        p = ctx.problem
        if (p.image_feats, p.depth, p.projection) != (feats.data_ptr(), depth.data_ptr(), proj.data_ptr()):
            # the saved tensors came back at other addresses (a saved-tensor hook moved them): describe them anew
            grid = torch.tensor(ctx.grid, dtype=torch.int32)  # host tensor: no synchronisation
            saved = (ctx.problem.saved_state, ctx.problem.saved_state_bytes)
            p, held = make_problem(depth, feats, proj, fsize, isize, roi, grid, spec, ctx.epsilon,
                                   ctx.depth_weight_threshold)  # `held` keeps the call's scratch alive until launched
            p.saved_state, p.saved_state_bytes = saved
        else:
            p.workspace = workspace(feats.device, torch.cuda.current_stream(feats.device).cuda_stream).data_ptr()
        flags = 0
        if ctx.needs_input_grad[1]:
            flags |= _lib.BWD_FEATS
        if ctx.needs_input_grad[0]:
            flags |= _lib.BWD_DEPTH
        if spec.legacy_depth_grad:
            flags |= _lib.BWD_LEGACY_DEPTH
        if spec.deterministic:
            flags |= _lib.BWD_DETERMINISTIC
        grad_feats = grad_depth = None
        if flags & (_lib.BWD_FEATS | _lib.BWD_DEPTH):
            go = _on(out_grad, feats.device, _out_dtype(spec, feats))
            lib = _lib.load()
            if flags & _lib.BWD_FEATS:
                grad_feats = torch.empty_like(feats)
            if flags & _lib.BWD_DEPTH:
                grad_depth = torch.empty_like(depth)
            nbytes = lib.fbev_backward_scratch_bytes(ctypes.byref(p), flags)
            scratch = torch.empty(nbytes, dtype=torch.uint8, device=feats.device) if nbytes else None
            with _on_device(feats.device):
                stream = torch.cuda.current_stream(feats.device).cuda_stream
                rc = lib.fbev_backward(
                    ctypes.byref(p), go.data_ptr(),
                    grad_feats.data_ptr() if grad_feats is not None else None,
                    grad_depth.data_ptr() if grad_depth is not None else None,
                    scratch.data_ptr() if scratch is not None else None, nbytes, flags, stream)
            _lib.check(rc, "fbev_backward")
            if grad_depth is not None and grad_depth.dtype != ctx.in_dtypes[0]:
                grad_depth = grad_depth.to(ctx.in_dtypes[0])
            if grad_feats is not None and grad_feats.dtype != ctx.in_dtypes[1]:
                grad_feats = grad_feats.to(ctx.in_dtypes[1])
        return (grad_depth, grad_feats, None, None, None, None, None, None, None, None, None, None, None, None)


def flash_bevpool(image_feats, depth_params, projection_matrices, feature_size, image_size, roi_range, grid_size,
                  depth_distribution=0, use_shared_memory=True, optimize_z_precompute=True, use_warp_kernel=False,
                  use_vectorized_load=False, epsilon=1e-6, depth_weight_threshold=1e-6, *, pool=None,
                  depth_bin_range=None, legacy_depth_grad=False, y_range=None, out_dtype=None, out=None,
                  host_row_chunks=0, save_lists=False, compact_rows=False, deterministic=False):
    """Fused BEV pooling; same arguments as the reference wrapper (flash_bevpool.py:139-178).

    Args:
        image_feats: [B,N,H,W,C] channels-last features (float32 / bfloat16 / float16).
        depth_params: [B,N,H,W,2] (mean, sigma) for ``depth_distribution`` 0 / 1, [B,N,H,W,D] probabilities
            for 2, or [B,N,H,W,D] logits for 3 (softmax over D folded into the operator and its backward).
        projection_matrices: [B,N,3,4] or [B,N,4,4].
        feature_size: [B,N,2] int (h, w).  image_size: [2] int (height, width).
        roi_range: [6] xmin,xmax,ymin,ymax,zmin,zmax.  grid_size: [3] int grid_x, grid_y, grid_z.
        depth_distribution: 0 gaussian, 1 laplace, 2 categorical, 3 categorical from logits (2 and 3 need
            ``depth_bin_range``).
        pool: "mean" (default for 0/1, the reference's) or "sum" (default for 2).
        depth_bin_range: (first bin edge, bin width) of the categorical mode.
        legacy_depth_grad: parametric modes only; reproduce the reference CUDA kernel's depth gradient.
        deterministic: backward with bitwise reproducible gradients (fixed-point sums instead of float sums in
            arrival order; 1.4 to 1.8 times the default backward's time on the benchmark shapes, same tolerances; at
            most 32 cameras).  The forward is reproducible anyway.
        y_range: (begin, end) BEV rows to compute; the other rows of the output are zero.
        compact_rows: with ``y_range``: the result (and the upstream gradient of its backward) holds only those
            rows, [B, end - begin, X, C]: a row shard that stays a shard.
        out_dtype: None (output in the feature dtype) or torch.float32 (what the reference returns for
            any input dtype).
        out: result buffer to fill and return instead of a new tensor: on the device, or page-locked host
            memory, which the kernel then writes directly (inference only; the caller synchronises the stream
            before reading it).
        host_row_chunks: with a host ``out``: 0 lets the kernel store to it over the bus; 1..16 computes that
            many bands of rows into a device buffer and copies each band while the next is computed.
        save_lists: True makes a forward whose inputs require gradients keep the row records and sample lists it
            builds (device memory of about 24 bytes per (cell, camera, height bin), freed with the graph) for the
            backward, which otherwise rebuilds them as the reference does.  Off by default: measured on the
            benchmark shape it moves 9 us into the forward to take 3 us out of the backward.
    Returns:
        BEV features [B,Y,X,C] in the dtype of ``image_feats`` (or float32, see ``out_dtype``).
    """
    refuse_tangents(image_feats, depth_params)
    spec = DepthSpec(depth_distribution, pool=pool, depth_bin_range=depth_bin_range,
                     legacy_depth_grad=legacy_depth_grad, y_range=y_range, out_dtype=out_dtype, out=out,
                     host_row_chunks=host_row_chunks, save_lists=save_lists, compact_rows=compact_rows,
                     deterministic=deterministic)
    if not (torch.is_grad_enabled() and (image_feats.requires_grad or depth_params.requires_grad)):
        return _forward(depth_params, image_feats, projection_matrices, feature_size, image_size, roi_range, grid_size,
                        spec, epsilon, depth_weight_threshold, False)[0]
    return FlashBEVPool.apply(depth_params, image_feats, projection_matrices, feature_size, image_size, roi_range,
                              grid_size, spec, use_shared_memory, optimize_z_precompute, use_warp_kernel,
                              use_vectorized_load, epsilon, depth_weight_threshold)


def debug_indices(image_feats, depth_params, projection_matrices, feature_size, image_size, roi_range, grid_size,
                  depth_distribution=0, epsilon=1e-6, depth_weight_threshold=1e-6, *, pool=None,
                  depth_bin_range=None):
    """Integer decisions of every (b, n, y, x, z) candidate, for bit-exact comparison with a CPU check.

    Returns dict(u0, v0, kbin: int32 [B,N,Y,X,Z]; valid: uint8 [B,N,Y,X,Z]; count: int32 [B,Y,X]).
    """
    spec = DepthSpec(depth_distribution, pool=pool, depth_bin_range=depth_bin_range)
    p, keep = make_problem(depth_params, image_feats, projection_matrices, feature_size, image_size, roi_range,
                           grid_size, spec, epsilon, depth_weight_threshold)
    dev = keep[0].device
    shp = (p.B, p.N, p.Y, p.X, p.Z)
    u0 = torch.empty(shp, dtype=torch.int32, device=dev)
    v0 = torch.empty_like(u0)
    kb = torch.empty_like(u0)
    va = torch.empty(shp, dtype=torch.uint8, device=dev)
    cnt = torch.empty((p.B, p.Y, p.X), dtype=torch.int32, device=dev)
    with torch.cuda.device(dev):
        rc = _lib.load().fbev_debug_indices(ctypes.byref(p), u0.data_ptr(), v0.data_ptr(), kb.data_ptr(),
                                            va.data_ptr(), cnt.data_ptr(), torch.cuda.current_stream().cuda_stream)
    _lib.check(rc, "fbev_debug_indices")
    return {"u0": u0, "v0": v0, "kbin": kb, "valid": va, "count": cnt}


def forward_with_count(image_feats, depth_params, projection_matrices, feature_size, image_size, roi_range,
                       grid_size, depth_distribution=0, epsilon=1e-6, depth_weight_threshold=1e-6, *, pool=None,
                       depth_bin_range=None, y_range=None, out_dtype=None):
    """Forward without autograd that also returns the per-cell count of accepted samples [B,Y,X]."""
    spec = DepthSpec(depth_distribution, pool=pool, depth_bin_range=depth_bin_range, y_range=y_range,
                     out_dtype=out_dtype)
    p, keep = make_problem(depth_params, image_feats, projection_matrices, feature_size, image_size, roi_range,
                           grid_size, spec, epsilon, depth_weight_threshold)
    dev = keep[0].device
    out = torch.zeros((p.B, p.Y, p.X, p.C), dtype=_out_dtype(spec, keep[0]), device=dev)
    cnt = torch.zeros((p.B, p.Y, p.X), dtype=torch.int32, device=dev)
    with torch.cuda.device(dev):
        rc = _lib.load().fbev_forward(ctypes.byref(p), out.data_ptr(), cnt.data_ptr(),
                                      torch.cuda.current_stream().cuda_stream)
    _lib.check(rc, "fbev_forward")
    return out, cnt
