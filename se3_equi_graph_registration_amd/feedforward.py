"""The gated feed-forward block: ``gated_feed_forward`` (HIP forward and backward, csrc/feed_forward.hip) and ``GatedFeedForward``, the
layer with its parameters.  Stands beside the two-Linear MLPs of ``E_GCL``, ``SO3TensorProductLayer`` and ``PointNetLayer``, which are
compiled for their narrow widths."""
from __future__ import annotations

from torch import nn

from .ops import autocast_type, context_ops, need_float

ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2}      # EQUIGSPR_ACT_*


def gated_feed_forward(x, w_gate, w_up, w_down, b_gate=None, b_up=None, b_down=None, *, activation="silu"):
    """``(act(x w_gate^T + b_gate) * (x w_up^T + b_up)) w_down^T + b_down`` -> ``[..., out]``.

    ``x [..., width]``, ``w_gate`` and ``w_up [hidden, width]``, ``w_down [out, hidden]`` (the layout of ``nn.Linear``), biases optional:
    float32, bfloat16 or float16, all alike, on one device (tensors that are not contiguous are copied).  ``activation``: "silu", "gelu"
    (exact) or "relu".  Products accumulate in fp32; the hidden layer is held in the inputs' dtype between the two products, as are the
    projections' gradients in the backward.  In float16 the hidden layer must stay within that type's range; the projections' gradients are
    held relative to the largest output gradient, must stay within 2^12 times it and lose bits below 2^-10 of it.  The backward keeps both
    projections in float32.  In float32 an infinity in a product's operand gives NaN.  Up to 8 388 480 rows a call.  Differentiable once in
    every tensor (reverse mode; tangents are refused); bitwise reproducible (no atomics)."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"gated_feed_forward: activation {activation!r}, expected one of {sorted(ACTIVATIONS)}")
    need_float(x, "x")
    if x.dim() < 1:
        raise RuntimeError("x: expected [..., width], got a scalar")
    for t, name in ((w_gate, "w_gate"), (w_up, "w_up"), (w_down, "w_down")):
        need_float(t, name, like=x, ndim=2)
    hidden, width = w_gate.shape
    out = w_down.shape[0]
    if x.shape[-1] != width or w_up.shape != w_gate.shape or w_down.shape[1] != hidden or min(hidden, width, out) < 1:
        raise RuntimeError(f"gated_feed_forward: x {tuple(x.shape)}, w_gate {tuple(w_gate.shape)}, w_up {tuple(w_up.shape)} and w_down "
                           f"{tuple(w_down.shape)} do not belong together")
    for t, name, n in ((b_gate, "b_gate", hidden), (b_up, "b_up", hidden), (b_down, "b_down", out)):
        if t is not None and need_float(t, name, like=x, ndim=1).shape[0] != n:
            raise RuntimeError(f"{name}: expected [{n}], got {tuple(t.shape)}")
    args = [x.reshape(-1, width).contiguous(), w_gate.contiguous(), w_up.contiguous(), w_down.contiguous()]
    args += [None if t is None else t.contiguous() for t in (b_gate, b_up, b_down)]
    return context_ops().gated_feed_forward(*args, ACTIVATIONS[activation]).view(*x.shape[:-1], out)


class GatedFeedForward(nn.Module):
    """``gated_feed_forward`` with its parameters: ``gate`` and ``up`` (width -> hidden), ``down`` (hidden -> width).  Under ``torch.autocast``
    the block runs in its type, as ``nn.Linear`` does."""

    def __init__(self, width, hidden, activation="silu", bias=True):
        super().__init__()
        if activation not in ACTIVATIONS:
            raise ValueError(f"GatedFeedForward: activation {activation!r}, expected one of {sorted(ACTIVATIONS)}")
        self.activation = activation
        self.gate, self.up = nn.Linear(width, hidden, bias=bias), nn.Linear(width, hidden, bias=bias)
        self.down = nn.Linear(hidden, width, bias=bias)

    def forward(self, x):
        args = [x, self.gate.weight, self.up.weight, self.down.weight, self.gate.bias, self.up.bias, self.down.bias]
        dtype = autocast_type()
        if dtype is not None:
            args = [None if t is None else t.to(dtype) for t in args]
        return gated_feed_forward(*args, activation=self.activation)
