"""Attention between the points of clouds: ``cloud_attention`` (HIP forward and backward, csrc/attention.hip and attention_bwd.hip) and
``CloudAttention``, the layer with its projections.

Beside the local aggregation over k-NN neighbours (``EGNN``, ``GraphConvolution``, ``PointNetLayer``) this lets every point look at all
points of its own cloud or of the other one.  No counterpart in the reference (its ``CrossAttentionPoseRegression`` holds no attention)."""
from __future__ import annotations

import math

import torch
from torch import nn

from .ops import autocast_type, context_ops, need_float


def _rows(t):
    """The kernels walk rows of unit stride, points and heads less than 2^31 / 128 bytes apart; any other stride is taken as it is."""
    n, m = t.stride(1) if t.shape[1] > 1 else 0, t.stride(2) if t.shape[2] > 1 else 0
    return t if (n + m) * 128 * t.element_size() < 1 << 31 and (t.shape[-1] == 1 or t.stride(-1) == 1) else t.contiguous()


def _need_lens(t, name, q):
    if t is None:
        return None
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor, got {type(t)}")
    if t.device != q.device or t.dtype != torch.int32 or t.shape != (q.shape[0],):
        raise RuntimeError(f"{name}: expected int32 [{q.shape[0]}] on {q.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.contiguous()


def cloud_attention(q, k, v, *, q_lens=None, kv_lens=None, key_mask=None, causal=False, scale=None):
    """``softmax(scale q k^T) v`` per head -> ``[B, Nq, H, D]``, contiguous, of the inputs' dtype.

    ``q [B, Nq, H, D]``, ``k`` and ``v [B, Nk, Hk, D]``: float32, bfloat16 or float16 on one device, ``1 <= D <= 128``, any strides
    (a last dimension that is not dense is copied).  ``H`` is a multiple of ``Hk``: query head ``h`` reads key head ``h // (H // Hk)``.
    ``q_lens`` / ``kv_lens`` (int32 ``[B]``, on the device): points of every sample that exist (clamped to ``[0, Nq]`` / ``[0, Nk]``).
    ``key_mask`` (bool ``[B, Nk]``): False hides a key.  ``causal``: point ``i`` sees the keys up to ``i + kv_len - q_len``.
    ``scale``: positive, default ``D ** -0.5``.

    A point without a visible key, and a point behind ``q_lens``, gives zeros and takes no gradient.  Keys hidden by ``kv_lens`` or
    ``key_mask`` are never used, whatever they hold, and their gradients are zero; a key that ``causal`` hides from some points only has
    weight zero there, so its values must be finite.  A NaN that a point sees reaches its output and every gradient of its keys; in float32
    an infinity in k or v does so as NaN.  Differentiable once in q, k and v (reverse mode; tangents are refused); bitwise reproducible (no
    atomics).  Scores, probabilities' sums and gradients' sums are fp32."""
    need_float(q, "q", ndim=4)
    need_float(k, "k", like=q, ndim=4)
    need_float(v, "v", like=q, ndim=4)
    b, nq, h, d = q.shape
    if k.shape != v.shape or k.shape[0] != b or k.shape[3] != d:
        raise RuntimeError(f"cloud_attention: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not belong together")
    if k.shape[2] < 1 or h < 1 or h % k.shape[2]:
        raise RuntimeError(f"cloud_attention: {h} heads are not a multiple of {k.shape[2]} key heads")
    if not 1 <= d <= 128:
        raise NotImplementedError(f"cloud_attention: head dim {d}, the HIP kernels take 1..128")
    scale = d ** -0.5 if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError("cloud_attention: scale must be positive and finite")
    q_lens, kv_lens = _need_lens(q_lens, "q_lens", q), _need_lens(kv_lens, "kv_lens", q)
    if key_mask is not None:
        if not isinstance(key_mask, torch.Tensor):
            raise TypeError(f"key_mask: expected a torch.Tensor, got {type(key_mask)}")
        if key_mask.device != q.device or key_mask.dtype != torch.bool or key_mask.shape != (b, k.shape[1]):
            raise RuntimeError(f"key_mask: expected bool [{b}, {k.shape[1]}] on {q.device}, got {key_mask.dtype} {tuple(key_mask.shape)} "
                               f"on {key_mask.device}")
        if key_mask.shape[1] > 1 and key_mask.stride(1) != 1:
            key_mask = key_mask.contiguous()
    return context_ops().cloud_attention(_rows(q), _rows(k), _rows(v), q_lens, kv_lens, key_mask, bool(causal), scale)


class CloudAttention(nn.Module):
    """Multi-head attention over point features: ``forward(h [B, N, width], other=None)`` attends to ``other [B, M, width]`` (default: ``h``
    itself).  ``kv_heads`` < ``num_heads`` shares keys and values between groups of heads.  The projections carry no bias."""

    def __init__(self, width, num_heads=4, kv_heads=None):
        super().__init__()
        kv_heads = num_heads if kv_heads is None else kv_heads
        if num_heads < 1 or width % num_heads or kv_heads < 1 or num_heads % kv_heads:
            raise ValueError("CloudAttention: width must be a multiple of num_heads, num_heads a multiple of kv_heads")
        if width // num_heads > 128:
            raise NotImplementedError("CloudAttention: the HIP kernels take head dims up to 128")
        self.width, self.num_heads, self.kv_heads, self.head_dim = width, num_heads, kv_heads, width // num_heads
        self.to_q = nn.Linear(width, width, bias=False)
        self.to_k = nn.Linear(width, kv_heads * self.head_dim, bias=False)
        self.to_v = nn.Linear(width, kv_heads * self.head_dim, bias=False)
        self.to_out = nn.Linear(width, width, bias=False)

    def forward(self, h, other=None, *, q_lens=None, kv_lens=None, key_mask=None):
        other = h if other is None else other
        b, n, _ = h.shape
        dtype = autocast_type()
        # under autocast the casts are made here: its own keep a weight's copy for as long as the context lasts, past the optimizer's update
        # when the context is around a loop, and out of reach of a captured step
        project = lambda layer, x: layer(x) if dtype is None else nn.functional.linear(x, layer.weight.to(dtype))  # noqa: E731
        if dtype is not None:
            h, other = h.to(dtype), other.to(dtype)
        q = project(self.to_q, h).view(b, n, self.num_heads, self.head_dim)
        k = project(self.to_k, other).view(b, other.shape[1], self.kv_heads, self.head_dim)
        v = project(self.to_v, other).view(b, other.shape[1], self.kv_heads, self.head_dim)
        out = cloud_attention(q, k, v, q_lens=q_lens, kv_lens=kv_lens, key_mask=key_mask)
        return project(self.to_out, out.view(b, n, self.width))
