"""CPU checks of the query operators: refusals in Python and status codes of the C ABI (no kernel is launched here)."""
import ctypes

import pytest
import torch

from flashbev_b200 import _lib, add_rms_norm, cross_attention, rotary_axes


def test_struct_layout_matches_the_header():
    assert ctypes.sizeof(_lib.FbevAttention) == 184 and ctypes.sizeof(_lib.FbevRotary) == 1248
    assert _lib.FbevAttention.q_stride.offset == 40 and _lib.FbevAttention.q.offset == 120
    assert _lib.FbevRotary.x.offset == 80 and _lib.FbevRotary.pair_turns.offset == 96


def test_operators_refuse_cpu_tensors():
    q = torch.zeros(1, 2, 2, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        cross_attention(q, q, q)
    with pytest.raises(RuntimeError, match="CUDA"):
        rotary_axes(q, torch.zeros(2, 1), (4,))
    with pytest.raises(RuntimeError, match="CUDA"):
        add_rms_norm(q)


def _attention():
    p = _lib.FbevAttention()
    p.struct_size = ctypes.sizeof(p)
    p.dtype = _lib.BF16
    p.B, p.Lq, p.Lk, p.Hq, p.Hkv, p.D, p.scale = 2, 5, 7, 4, 2, 64, 0.125
    p.q_stride[:], p.k_stride[:], p.v_stride[:] = (1280, 256, 64), (896, 128, 64), (896, 128, 64)
    p.q = p.k = p.v = 4096  # never dereferenced: validation fails first in every case below
    p.workspace, p.workspace_bytes = 1 << 20, 1 << 40
    return p


def test_attention_status_codes():
    lib = _lib.load()
    fwd = lambda p: lib.fbev_cross_attention(ctypes.byref(p), 4096, None, None)  # noqa: E731
    bwd = lambda p: lib.fbev_cross_attention_grad(ctypes.byref(p), 4096, 4096, 4096, 4096, 4096, 4096, None)  # noqa: E731
    assert lib.fbev_cross_attention(None, 4096, None, None) == 1
    for field, value, code in (("struct_size", 8, 2), ("dtype", 7, 4), ("B", -1, 3), ("Hkv", 3, 3), ("Hkv", 0, 3), ("D", 0, 3),
                               ("D", 129, 3), ("Lq", 1 << 30, 7), ("key_lengths", 6, 6), ("status", 2, 6), ("q", 4097, 6)):
        p = _attention()
        setattr(p, field, value)
        assert fwd(p) == code and bwd(p) == code, (field, value)
        assert lib.fbev_cross_attention_lse_count(ctypes.byref(p)) == 0
        assert lib.fbev_cross_attention_workspace_bytes(ctypes.byref(p), 1) == 0
    p = _attention()
    assert lib.fbev_cross_attention_lse_count(ctypes.byref(p)) == 2 * 2 * 12  # ten rows, padded to a multiple of four
    p.k = None
    assert fwd(p) == 1 and bwd(p) == 1
    p = _attention()
    assert lib.fbev_cross_attention(ctypes.byref(p), None, None, None) == 1
    assert lib.fbev_cross_attention(ctypes.byref(p), 4097, None, None) == 6
    assert lib.fbev_cross_attention(ctypes.byref(p), 4096, 4100, None) == 6           # statistics: 16 bytes
    assert lib.fbev_cross_attention_grad(ctypes.byref(p), 4096, 4096, 4096, 4096, 4096, None, None) == 1
    assert lib.fbev_cross_attention_grad(ctypes.byref(p), 4096, None, 4096, 4096, 4096, 4096, None) == 1
    assert lib.fbev_cross_attention_grad(ctypes.byref(p), 4096, 4096, 4096, None, None, None, None) == 0
    assert lib.fbev_cross_attention_workspace_bytes(ctypes.byref(p), 1) > 0
    for value in (None, (1 << 20) + 8):
        p = _attention()
        p.workspace = value
        assert bwd(p) == 8
    p = _attention()
    p.workspace_bytes = 16
    assert bwd(p) == 8
    for field in ("B", "Lq"):
        p = _attention()
        setattr(p, field, 0)
        assert lib.fbev_cross_attention(ctypes.byref(p), None, None, None) == 0


def test_rotary_and_norm_status_codes():
    lib = _lib.load()

    def rotary(**kw):
        p = _lib.FbevRotary()
        p.struct_size = ctypes.sizeof(p)
        p.dtype, p.B, p.L, p.H, p.D, p.pairs, p.axes, p.x, p.positions = _lib.F32, 1, 2, 2, 16, 8, 2, 4096, 4096
        out = kw.pop("out", 4096)
        axis = kw.pop("axis", 0)
        p.pair_axis[3] = axis
        for n, value in kw.items():
            setattr(p, n, value)
        return lib.fbev_rotary_axes(ctypes.byref(p), out, None)

    assert lib.fbev_rotary_axes(None, 4096, None) == 1
    for kw, code in (({"struct_size": 4}, 2), ({"dtype": 3}, 4), ({"pos_dtype": 3}, 4), ({"D": 257}, 3), ({"pairs": 9}, 3),
                     ({"pairs": -1}, 3), ({"axes": 0}, 3), ({"axes": 9}, 3), ({"axis": 2}, 3), ({"out": None}, 1),
                     ({"x": None}, 1), ({"positions": None}, 1), ({"x": 4098}, 6), ({"positions": 4098}, 6),
                     ({"L": 0, "x": None}, 0)):
        assert rotary(**kw) == code, kw
    norm = lambda dtype=0, rows=4, C=16, x=4096, r=None, w=None, y=4096, h=None, s=None: lib.fbev_add_rms_norm(  # noqa: E731
        dtype, rows, C, 1e-6, x, r, w, y, h, s, None)
    for kw, code in (({"dtype": 5}, 4), ({"rows": -1}, 3), ({"C": 0}, 3), ({"C": (1 << 20) + 1}, 7), ({"x": None}, 1),
                     ({"y": None}, 1), ({"x": 4097}, 6), ({"r": 4098}, 6), ({"s": 2}, 6), ({"rows": 0, "x": None}, 0)):
        assert norm(**kw) == code, kw
    assert lib.fbev_add_rms_norm_e4m3(0, 4, 16, 1e-6, 4096, None, None, 4096, None, None, None) == 1
    grad = lambda h=4096, gx=4096, gw=4096, ws=4096, n=1 << 30: lib.fbev_add_rms_norm_grad(  # noqa: E731
        0, 4, 16, h, 4096, None, 4096, None, gx, gw, ws, n, None)
    assert grad(h=None) == 1 and grad(ws=None) == 8 and grad(n=8) == 8 and grad(ws=4100) == 8
    assert grad(gx=None, gw=None) == 0
    assert lib.fbev_add_rms_norm_grad_workspace_bytes(4, 16, 1) == 256 and lib.fbev_add_rms_norm_grad_workspace_bytes(4, 16, 0) == 0


def test_camera_attention_is_optional_and_checks_its_sizes():
    from flashbev_b200 import CameraAttention, SamplingVT
    grid = {"x": [-4.0, 4.0, 1.0], "y": [-2.0, 2.0, 1.0], "z": [-4.0, 2.0, 1.0], "depth": [1.0, 60.0, 1.0]}
    plain = SamplingVT(grid, (128, 352), in_channels=8, out_channels=16)
    assert plain.camera_attention is None and not any("attention" in k for k in plain.state_dict())
    m = SamplingVT(grid, (128, 352), in_channels=8, out_channels=16, attention_heads=2)
    cells = m.camera_attention.cell_positions
    assert cells.shape == (4 * 8, 2) and cells[0].tolist() == [-1.5, -3.5] and cells[-1].tolist() == [1.5, 3.5]
    assert set(plain.state_dict()) < set(m.state_dict())
    for channels, heads, key_heads in ((16, 3, None), (6, 2, None), (256, 1, None), (16, 4, 3), (16, 0, None)):
        with pytest.raises(ValueError):
            CameraAttention(channels, 8, heads, torch.zeros(4, 2), key_heads=key_heads)


def test_scores_have_a_finite_factor():
    lib = _lib.load()
    for scale in (float("nan"), float("inf"), -float("inf"), 2e30, -2e30):
        p = _attention()
        p.scale = scale
        assert lib.fbev_cross_attention(ctypes.byref(p), 4096, None, None) == 7
        assert lib.fbev_cross_attention_grad(ctypes.byref(p), 4096, 4096, 4096, 4096, 4096, 4096, None) == 7
