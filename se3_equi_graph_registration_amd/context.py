"""``CloudContext``: blocks that let the points of two clouds see each other, between the EGNN and the pose head
(``CrossAttentionPoseRegression(egnn, ..., context=CloudContext(32))``).

A layer is self-attention within every cloud, attention to the other cloud of the pair, and a gated feed-forward block; between the three
runs ``residual_norm``: the norm behind the block, its residual scale, the addition and the norm before the next one in one launch.  No
counterpart in the reference, whose pair model compares the two clouds only in its head."""
from __future__ import annotations

import torch
from torch import nn

from .attention import CloudAttention
from .feedforward import GatedFeedForward
from .norms import ResidualNorm
from .ops import need_float


class CloudContext(nn.Module):
    """``forward(h [2, B, N, width], valid=None) -> [2, B, N, width]``: ``h[0]`` / ``h[1]`` the point features of the source / target clouds.
    ``valid`` (bool ``[2, B, N]``): points that exist; the others are not attended to (their own rows are computed all the same, so they
    must be finite: zeros, not NaN).  ``residual_scale`` starts the blocks near the identity.

    The blocks run in the type of their parameters (``CloudContext(...).bfloat16()`` behind an fp32 EGNN), or, their products, in that of
    ``torch.autocast``; the result has the type of ``h``.  (``train.make_optimizer`` keeps every parameter in fp32: train in 16 bits under
    autocast.)"""

    def __init__(self, width, n_layers=1, num_heads=4, hidden=None, kind="layer", activation="silu", residual_scale=0.1, device="cuda:0"):
        super().__init__()
        if n_layers < 1:
            raise ValueError("CloudContext: n_layers must be positive")
        hidden = 4 * width if hidden is None else hidden
        self.width, self.n_layers = width, n_layers
        self.first = ResidualNorm(width, kind, post=False)
        self.self_attention = nn.ModuleList([CloudAttention(width, num_heads) for _ in range(n_layers)])
        self.cross_attention = nn.ModuleList([CloudAttention(width, num_heads) for _ in range(n_layers)])
        self.feed_forward = nn.ModuleList([GatedFeedForward(width, hidden, activation, bias=False) for _ in range(n_layers)])
        # behind every block, and (but for the last) before the next one
        self.steps = nn.ModuleList([ResidualNorm(width, kind, pre=i + 1 < 3 * n_layers, residual_scale=residual_scale) for i in range(3 * n_layers)])
        self.to(device)

    def forward(self, h, valid=None):
        if h.dim() != 4 or h.shape[0] != 2 or h.shape[3] != self.width:
            raise RuntimeError(f"CloudContext: expected h [2, B, N, {self.width}], got {tuple(h.shape)}")
        need_float(h, "h")
        _, b, n, c = h.shape
        if valid is not None and (valid.dtype != torch.bool or valid.shape != (2, b, n)):
            raise RuntimeError(f"valid: expected bool [2, {b}, {n}], got {valid.dtype} {tuple(valid.shape)}")
        mask = None if valid is None else valid.reshape(2 * b, n)
        other_mask = None if valid is None else valid.flip(0).reshape(2 * b, n)
        x = h.reshape(2 * b, n, c).to(self.first.pre_weight.dtype)
        _, u = self.first(x)
        step = iter(self.steps)
        for i in range(self.n_layers):
            x, u = next(step)(x, self.self_attention[i](u, key_mask=mask))
            x, u = next(step)(x, self.cross_attention[i](u, torch.cat([u[b:], u[:b]]), key_mask=other_mask))
            x, u = next(step)(x, self.feed_forward[i](u))
        return x.view(2, b, n, c).to(h.dtype)
