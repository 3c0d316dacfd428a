"""``CameraAttention``: BEV cells attend to the cameras' tokens, on the operators of ``query_ops``.

A view transform samples, for each BEV cell, the few feature-map positions its voxel centres project to.  This block lets
every cell look at all positions of all cameras afterwards: one pre-norm attention block (and a small feed-forward) over
the pooled BEV features.  ``SamplingVT(attention_heads=n)`` appends it; with ``n = 0`` (the default) nothing of it exists
and the module is the reference's.  The reference (yokosyun/FlashBEV) has no counterpart.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from .query_ops import add_rms_norm, cross_attention, rotary_axes


class CameraAttention(nn.Module):
    """x [B,C,Y,X] -> x + attention(norm(x), tokens) -> + feed-forward(norm(.)), the same layout.

    Args:
        channels: C of the BEV features.  token_channels: channels of the camera features.
        heads: query heads; C must be a multiple, and the head width even and at most 128.
        key_heads: heads of keys and values, a divisor of ``heads`` (default: as many).
        cell_positions: [Y*X,2] coordinates (y, x) of the cells, in any unit; the rotary positions of the queries.
    The output projections start at zero, so the block starts as the identity.  Under ``torch.autocast`` the products and the
    attention run in its type, norms and residual in the type of the BEV features, which the result has too.
    """

    def __init__(self, channels, token_channels, heads, cell_positions, key_heads=None):
        super().__init__()
        key_heads = heads if key_heads is None else key_heads
        if heads < 1 or channels % heads != 0:
            raise ValueError(f"{channels} channels do not divide into {heads} heads")
        width = channels // heads
        if width % 2 or width > 128:
            raise ValueError(f"the head width must be even and at most 128, got {width}")
        if key_heads < 1 or heads % key_heads != 0:
            raise ValueError(f"the number of heads ({heads}) must be a multiple of the key heads ({key_heads})")
        self.heads, self.key_heads, self.width = heads, key_heads, width
        self.norm_attention = nn.Parameter(torch.ones(channels))
        self.norm_forward = nn.Parameter(torch.ones(channels))
        self.to_q = nn.Linear(channels, channels, bias=False)
        self.to_kv = nn.Linear(token_channels, 2 * key_heads * width, bias=False)
        self.to_out = nn.Linear(channels, channels, bias=False)
        self.widen = nn.Linear(channels, 2 * channels)
        self.narrow = nn.Linear(2 * channels, channels)
        for layer in (self.to_out, self.narrow):
            nn.init.zeros_(layer.weight)
        nn.init.zeros_(self.narrow.bias)
        # neither parameters nor buffers: they keep their type when the module's is changed
        self.cell_positions = cell_positions.to(device="cpu", dtype=torch.float32).contiguous()
        self._positions_on = {}

    def _sections(self, axes):
        """Even shares of the head's pairs, what is left over to the first axis."""
        pairs = self.width // 2
        return (pairs - pairs // axes * (axes - 1),) + (pairs // axes,) * (axes - 1)

    def _positions(self, device, cameras, h, w):
        """[Y*X,2] of the cells and [N*h*w,3] (camera, row, column) of the tokens, copied once per size and device."""
        key = (str(device), cameras, h, w)
        p = self._positions_on.get(key)
        if p is None:
            with torch.inference_mode(False):  # a call that trains keeps them for its backward
                n, y, x = torch.meshgrid(torch.arange(cameras), torch.arange(h), torch.arange(w), indexing="ij")
                tokens = torch.stack([n, y, x], dim=-1).view(-1, 3)
                p = self.cell_positions.to(device), tokens.to(device=device, dtype=torch.int32)
            self._positions_on[key] = p
        return p

    def forward(self, bev, features, cameras, camera_mask=None):
        """bev [B,C,Y,X] (channels-last strides are used as they are), features [B*cameras,Ct,h,w]; camera_mask [B,cameras]
        bool, False where a camera is missing.  The first call of a size copies positions to the device: make it before a
        graph is captured.  Before a training step is captured, let go of earlier results that still hold the parameters' graph:
        autograd ties a parameter to the stream of its first use."""
        B, C, Y, X = bev.shape
        h, w = features.shape[-2:]
        x = bev.permute(0, 2, 3, 1).reshape(B, Y * X, C)
        tokens = features.permute(0, 2, 3, 1).reshape(B, cameras * h * w, features.shape[1])
        cells, places = self._positions(bev.device, cameras, h, w)
        y, _ = add_rms_norm(x, None, self.norm_attention.to(x.dtype))
        q = rotary_axes(self.to_q(y).view(B, Y * X, self.heads, self.width), cells, self._sections(2))
        kv = self.to_kv(tokens).view(B, cameras * h * w, 2, self.key_heads, self.width)
        k = rotary_axes(kv[:, :, 0], places, self._sections(3))
        mask = None if camera_mask is None else camera_mask.repeat_interleave(h * w, dim=1)
        seen = self.to_out(cross_attention(q, k, kv[:, :, 1], key_mask=mask).flatten(2))
        # under autocast products come in its type, whatever the parameters'; the residual keeps the features' type
        y, x = add_rms_norm(seen.to(x.dtype), x, self.norm_forward.to(x.dtype))
        x = x + self.narrow(torch.nn.functional.gelu(self.widen(y))).to(x.dtype)
        return x.view(B, Y, X, C).permute(0, 3, 1, 2)
