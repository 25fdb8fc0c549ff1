"""The context operators' checks that need no GPU: CPU tensors are refused, and the C entries turn bad descriptions into error codes."""
import ctypes

import pytest
import torch

import se3_equi_graph_registration_amd as pk
from se3_equi_graph_registration_amd import _lib


def test_cpu_tensors_fail_loudly():
    t = torch.zeros(1, 4, 2, 8)
    with pytest.raises(RuntimeError, match="no CPU path"):
        pk.cloud_attention(t, t, t)
    with pytest.raises(RuntimeError, match="no CPU path"):
        pk.gated_feed_forward(torch.zeros(2, 8), torch.zeros(4, 8), torch.zeros(4, 8), torch.zeros(8, 4))
    with pytest.raises(RuntimeError, match="no CPU path"):
        pk.residual_norm(torch.zeros(2, 8), torch.zeros(2, 8))
    with pytest.raises(TypeError):
        pk.cloud_attention(None, t, t)


def test_modules_check_their_sizes():
    for bad in (lambda: pk.CloudAttention(33, 4), lambda: pk.CloudAttention(32, 4, 3), lambda: pk.GatedFeedForward(8, 8, "tanh"),
                lambda: pk.ResidualNorm(8, "batch"), lambda: pk.CloudContext(32, n_layers=0)):
        with pytest.raises(ValueError):
            bad()
    ctx = pk.CloudContext(32, n_layers=2, device="cpu")
    assert ctx.steps[-1].pre_weight is None and ctx.steps[0].pre_weight is not None
    assert set(n.split(".")[0] for n, _ in ctx.named_parameters()) == {"first", "self_attention", "cross_attention", "feed_forward", "steps"}
    with pytest.raises(RuntimeError):
        ctx(torch.zeros(2, 1, 4, 31))


def _attention(**over):
    one = _lib.AttentionTensor(16, 0, 0, 0)                                # never read: every call below is refused on the host
    d = dict(dtype=1, batch=2, nq=3, nk=4, heads=4, kv_heads=2, dim=16, causal=0, scale=0.25, q=one, k=one, v=one)
    d.update(over)
    return _lib.Attention(**d)


@pytest.mark.parametrize("over,code", [
    (dict(dtype=3), -1), (dict(batch=-1), -1), (dict(nq=-1), -1), (dict(heads=0), -1), (dict(heads=3), -1), (dict(dim=0), -2), (dict(dim=129), -2),
    (dict(scale=0.0), -1), (dict(scale=float("nan")), -1), (dict(scale=float("inf")), -1), (dict(nq=1 << 30), -2), (dict(batch=1 << 23), -2),
    (dict(q=_lib.AttentionTensor(None, 0, 0, 0)), -1), (dict(v=_lib.AttentionTensor(None, 0, 0, 0)), -1)])
def test_attention_entry_refuses(over, code):
    L = _lib.lib()
    d = _attention(**over)
    assert L.equigspr_attention_work_size(ctypes.byref(d)) == -1
    assert L.equigspr_attention_backward_work_size(ctypes.byref(d)) == -1
    assert L.equigspr_attention_forward(ctypes.byref(d), 16, None, None, None, None) == code
    assert L.equigspr_attention_backward(ctypes.byref(d), 16, None, 16, ctypes.byref(d.q), 16, None, None, None, None) == code
    assert L.equigspr_last_error()


def test_entries_refuse_null_pointers_and_bad_sizes():
    L = _lib.lib()
    d = _attention()
    assert L.equigspr_attention_forward(None, 16, None, None, None, None) == -1
    assert L.equigspr_attention_forward(ctypes.byref(d), None, None, None, None, None) == -1
    assert L.equigspr_attention_backward(ctypes.byref(d), 16, None, 16, None, 16, None, None, None, None) == -1
    long = _attention(nq=1, nk=100000, batch=1, kv_heads=4)
    assert L.equigspr_attention_work_size(ctypes.byref(long)) > 0
    assert L.equigspr_attention_forward(ctypes.byref(long), 16, None, None, None, None) == -1          # needs its workspace
    assert L.equigspr_attention_forward(ctypes.byref(_attention(batch=0)), None, None, None, None, None) == 0
    ff = dict(dtype=0, activation=0, rows=3, width=8, hidden=16, out=8, x=16, w_gate=16, w_up=16, w_down=16)
    for over in (dict(dtype=7), dict(activation=3), dict(rows=-1), dict(hidden=0), dict(x=None), dict(w_up=None)):
        f = _lib.GatedFeedForward(**{**ff, **over})
        assert L.equigspr_gated_feed_forward_forward(ctypes.byref(f), 16, 16, None, None, None) == -1
        assert L.equigspr_gated_feed_forward_work_size(ctypes.byref(f)) == -1
    f = _lib.GatedFeedForward(**ff)
    assert L.equigspr_gated_feed_forward_forward(ctypes.byref(f), None, 16, None, None, None) == -1
    assert L.equigspr_gated_feed_forward_backward(ctypes.byref(f), None, 16, 16, 16, 16, None, None) == -1
    rn = dict(dtype=0, width=8, rows=4, gate_rows=1, eps=1e-5, factor=1.0, x=16, f=16, pre_weight=16)
    for over, code in ((dict(dtype=9), -1), (dict(width=0), -2), (dict(width=8193), -2), (dict(rows=-1), -1), (dict(eps=-1.0), -1), (dict(x=None), -1),
                       (dict(gate=16, gate_rows=3), -1), (dict(f=None, scale=16), -1), (dict(f=None, pre_weight=None), -1)):
        r = _lib.ResidualNorm(**{**rn, **over})
        assert L.equigspr_residual_norm_forward(ctypes.byref(r), 16, 16, None) == code
        assert L.equigspr_residual_norm_backward_work_size(ctypes.byref(r)) == -1
    r = _lib.ResidualNorm(**rn)
    assert L.equigspr_residual_norm_forward(ctypes.byref(r), 16, None, None) == -1
    assert L.equigspr_residual_norm_backward(ctypes.byref(r), 16, 16, None, None, None) == -1
