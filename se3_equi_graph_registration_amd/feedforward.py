"""The gated feed-forward block: ``gated_feed_forward`` (HIP forward and backward, csrc/feed_forward.hip) and ``GatedFeedForward``, the
layer with its parameters.  Stands beside the two-Linear MLPs of ``E_GCL``, ``SO3TensorProductLayer`` and ``PointNetLayer``, which are
compiled for their narrow widths."""
from __future__ import annotations

import ctypes

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import DTYPE_CODES, _p, _stream, check_capture, need_float, on_device, wants_grad

ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2}      # EQUIGSPR_ACT_*


def _describe(x, w_gate, w_up, w_down, b_gate, b_up, b_down, act):
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    return _lib.GatedFeedForward(DTYPE_CODES[x.dtype], act, x.shape[0], x.shape[1], w_gate.shape[0], w_down.shape[0], ptr(x), ptr(w_gate),
                                 ptr(w_up), ptr(w_down), ptr(b_gate), ptr(b_up), ptr(b_down))


def _forward(x, w_gate, w_up, w_down, b_gate, b_up, b_down, act, training):
    L = _lib.lib()
    new = lambda *s: torch.empty(s, dtype=x.dtype, device=x.device)  # noqa: E731
    rows, hidden = x.shape[0], w_gate.shape[0]
    with on_device(x.device):
        desc = _describe(x, w_gate, w_up, w_down, b_gate, b_up, b_down, act)
        n = L.equigspr_gated_feed_forward_work_size(ctypes.byref(desc))
        work = torch.empty(n, dtype=torch.float32, device=x.device) if n > 0 else None
        y, h = new(rows, w_down.shape[0]), new(rows, hidden)
        zu = torch.empty(rows, 2 * hidden, dtype=torch.float32, device=x.device) if training else None
        _lib.check(L.equigspr_gated_feed_forward_forward(ctypes.byref(desc), _p(y), _p(h), _p(zu), _p(work), _stream()),
                   "gated_feed_forward_forward")
    return y, zu, h


class _FeedForwardFn(torch.autograd.Function):
    """``equigspr_gated_feed_forward_forward`` / ``_backward``; both projections and the hidden layer are kept."""

    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, b_gate, b_up, b_down, act):
        y, zu, h = _forward(x, w_gate, w_up, w_down, b_gate, b_up, b_down, act, True)
        ctx.save_for_backward(x, w_gate, w_up, w_down, zu, h)
        ctx.act = act
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        x, w_gate, w_up, w_down, zu, h = ctx.saved_tensors
        L = _lib.lib()
        need = ctx.needs_input_grad
        rows, width = x.shape
        hidden, out = w_gate.shape[0], w_down.shape[0]
        make = torch.empty if rows else torch.zeros
        new = lambda *s: make(s, dtype=x.dtype, device=x.device)  # noqa: E731
        with on_device(x.device):
            gy = gy.contiguous()
            desc = _describe(x, w_gate, w_up, w_down, None, None, None, ctx.act)
            gx = new(rows, width) if need[0] else None
            gw = new(2 * hidden, width) if need[1] or need[2] else None
            gd = new(out, hidden) if need[3] else None
            gb = new(2 * hidden) if need[4] or need[5] else None
            gbd = new(out) if need[6] else None
            dzu = new(rows, 2 * hidden)
            work = torch.empty(max(1, L.equigspr_gated_feed_forward_backward_work_size(ctypes.byref(desc))), dtype=torch.float32, device=x.device)
            ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
            grads = _lib.GatedFeedForwardGrads(ptr(gx), ptr(gw), ptr(gd), ptr(gb), ptr(gbd))
            _lib.check(L.equigspr_gated_feed_forward_backward(ctypes.byref(desc), _p(gy), _p(zu), _p(h), _p(dzu), _p(work), ctypes.byref(grads),
                                                              _stream()), "gated_feed_forward_backward")
        return (gx, gw[:hidden] if need[1] else None, gw[hidden:] if need[2] else None, gd, gb[:hidden] if need[4] else None,
                gb[hidden:] if need[5] else None, gbd, None)


def gated_feed_forward(x, w_gate, w_up, w_down, b_gate=None, b_up=None, b_down=None, *, activation="silu"):
    """``(act(x w_gate^T + b_gate) * (x w_up^T + b_up)) w_down^T + b_down`` -> ``[..., out]``.

    ``x [..., width]``, ``w_gate`` and ``w_up [hidden, width]``, ``w_down [out, hidden]`` (the layout of ``nn.Linear``), biases optional:
    float32, bfloat16 or float16, all alike, on one device (tensors that are not contiguous are copied).  ``activation``: "silu", "gelu"
    (exact) or "relu".  Products accumulate in fp32; the hidden layer is held in the inputs' dtype between the two products, as are the
    projections' gradients in the backward: in float16 they must stay within that type's range.  The backward keeps both projections in
    float32.  Differentiable once in every tensor; bitwise
    reproducible (no atomics)."""
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
    if wants_grad(*args):
        check_capture(*args)
        y = _FeedForwardFn.apply(*args, ACTIVATIONS[activation])
    else:
        y = _forward(*args, ACTIVATIONS[activation], False)[0]
    return y.view(*x.shape[:-1], out)


class GatedFeedForward(nn.Module):
    """``gated_feed_forward`` with its parameters: ``gate`` and ``up`` (width -> hidden), ``down`` (hidden -> width)."""

    def __init__(self, width, hidden, activation="silu", bias=True):
        super().__init__()
        if activation not in ACTIVATIONS:
            raise ValueError(f"GatedFeedForward: activation {activation!r}, expected one of {sorted(ACTIVATIONS)}")
        self.activation = activation
        self.gate, self.up = nn.Linear(width, hidden, bias=bias), nn.Linear(width, hidden, bias=bias)
        self.down = nn.Linear(hidden, width, bias=bias)

    def forward(self, x):
        return gated_feed_forward(x, self.gate.weight, self.up.weight, self.down.weight, self.gate.bias, self.up.bias, self.down.bias,
                                  activation=self.activation)
