"""The residual step between blocks: ``residual_norm`` (HIP forward and backward, csrc/residual_norm.hip) and ``ResidualNorm``, the layer
with its parameters.  The norm behind a block, its gate, the residual scale, the addition and the norm before the next block are one pass
over memory (the ``LayerNorm`` of ``E_GCL`` lives inside the edge kernels and is not reachable on its own)."""
from __future__ import annotations

import torch
from torch import nn

from .ops import autocast_type, context_ops, need_float

KINDS = ("layer", "rms")
_MAX_WIDTH = 8192


def residual_norm(x, f, pre_weight=None, pre_bias=None, *, post_weight=None, post_bias=None, gate=None, scale=None, kind="layer", eps=1e-5):
    """``z = norm(f) * post_weight + post_bias`` (``f`` itself without ``post_weight``), ``y = x + scale * gate * z``,
    ``u = norm(y) * pre_weight + pre_bias`` -> ``(y, u)``; without ``pre_weight`` ``u`` is None.  ``f=None``: ``y`` is ``x`` and only ``u`` is
    formed (the norm before the first block).

    ``x``, ``f [..., C]``: float32, bfloat16 or float16, alike, ``1 <= C <= 8192`` (copied if not contiguous).  ``kind``: "layer" (mean and
    spread) or "rms" (spread about zero, no mean).  ``gate`` (dtype of x): ``[C]``, one row per sample ``[B, C]`` for ``x [B, N, C]``, or the
    shape of ``x``.  ``scale``: a float or a tensor ``[C]``.  Weights, biases and a tensor scale are used in float32 (converted if not).
    Sums are fp32, the second norm takes ``y`` before its rounding.  Differentiable once in every tensor (reverse mode;
    tangents are refused); bitwise reproducible."""
    if kind not in KINDS:
        raise ValueError(f"residual_norm: kind {kind!r}, expected 'layer' or 'rms'")
    need_float(x, "x")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= _MAX_WIDTH:
        raise NotImplementedError(f"residual_norm: x {tuple(x.shape)}, the HIP kernels take widths 1..{_MAX_WIDTH}")
    eps = float(eps)
    if not 0 <= eps < float("inf"):
        raise ValueError("residual_norm: eps must be finite and not negative")
    c = x.shape[-1]
    if f is None:
        if pre_weight is None or any(t is not None for t in (post_weight, post_bias, gate, scale)):
            raise ValueError("residual_norm: without f there is only the norm before the next block (pre_weight, pre_bias)")
    elif need_float(f, "f", like=x).shape != x.shape:
        raise RuntimeError(f"f: expected {tuple(x.shape)}, got {tuple(f.shape)}")
    if (pre_bias is not None and pre_weight is None) or (post_bias is not None and post_weight is None):
        raise ValueError("residual_norm: a norm's bias needs its weight")
    rows = x.numel() // c
    gate_rows = max(rows, 1)
    if gate is not None:
        need_float(gate, "gate", like=x)
        if gate.shape == x.shape:
            gate_rows = 1
        elif x.dim() == 3 and gate.shape == (x.shape[0], c):
            gate_rows = max(x.shape[1], 1)
        elif gate.shape != (c,):
            raise RuntimeError(f"gate: expected [{c}], [B, {c}] for x [B, N, {c}], or the shape of x, got {tuple(gate.shape)}")
        gate = gate.contiguous()
    factor = 1.0
    if scale is not None and not isinstance(scale, torch.Tensor):
        factor, scale = float(scale), None
    params = []
    for t, name in ((pre_weight, "pre_weight"), (pre_bias, "pre_bias"), (post_weight, "post_weight"), (post_bias, "post_bias"), (gate, "gate"), (scale, "scale")):
        if t is not None and name != "gate":
            if need_float(t, name).shape != (c,) or t.device != x.device:
                raise RuntimeError(f"{name}: expected [{c}] on {x.device}, got {tuple(t.shape)} on {t.device}")
            t = t.float().contiguous()
        params.append(t)
    y, u = context_ops().residual_norm(x.contiguous(), None if f is None else f.contiguous(), *params, kind == "rms", eps, factor, gate_rows)
    return (x if f is None else y), (None if pre_weight is None else u)


class ResidualNorm(nn.Module):
    """``residual_norm`` with its parameters: ``forward(x, f=None, gate=None) -> (y, u)``.  ``post`` / ``pre``: the norm behind the block and
    the one before the next; ``residual_scale``: start value of a trainable scale per channel (None: no scale).  In the first step of a
    stack (``f=None``) the norm behind a block, the gate and the scale play no part.  Under ``torch.autocast`` ``f`` and ``gate`` may be of
    another type than ``x`` and are taken in that of ``x``."""

    def __init__(self, width, kind="layer", post=True, pre=True, residual_scale=None, eps=1e-5):
        super().__init__()
        if kind not in KINDS:
            raise ValueError(f"ResidualNorm: kind {kind!r}, expected 'layer' or 'rms'")
        if not 1 <= width <= _MAX_WIDTH:
            raise NotImplementedError(f"ResidualNorm: the HIP kernels take widths 1..{_MAX_WIDTH}")
        self.kind, self.eps = kind, eps
        weight = lambda on, v: nn.Parameter(torch.full((width,), float(v))) if on else None  # noqa: E731
        self.pre_weight, self.pre_bias = weight(pre, 1), weight(pre and kind == "layer", 0)
        self.post_weight, self.post_bias = weight(post, 1), weight(post and kind == "layer", 0)
        self.scale = weight(residual_scale is not None, residual_scale or 0)

    def forward(self, x, f=None, gate=None):
        if f is None:
            return residual_norm(x, None, self.pre_weight, self.pre_bias, kind=self.kind, eps=self.eps)
        if autocast_type() is not None:
            f, gate = f.to(x.dtype), None if gate is None else gate.to(x.dtype)
        return residual_norm(x, f, self.pre_weight, self.pre_bias, post_weight=self.post_weight, post_bias=self.post_bias, gate=gate,
                             scale=self.scale, kind=self.kind, eps=self.eps)
