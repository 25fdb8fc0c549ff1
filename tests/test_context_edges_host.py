"""More checks of the context operators that need no GPU: what the C entries make of descriptions at the ends of their types."""
import ctypes

import pytest

from se3_equi_graph_registration_amd import _lib
from tests.test_context_host import _attention


@pytest.mark.parametrize("point,head", [(1 << 57, 0), (0, 1 << 57), (1 << 56, 1 << 56), (1 << 62, 1 << 62), ((1 << 31) // 256, 0), (-1, 0), (0, -1)])
def test_attention_strides_out_of_range_are_refused(point, head):
    """Points or heads further apart than the kernels' 32-bit offsets reach, also where 128 times the stride wraps around 64 bits."""
    L = _lib.lib()
    far = _lib.AttentionTensor(16, 0, point, head)
    for name in "qkv":
        d = _attention(**{name: far})
        assert L.equigspr_attention_work_size(ctypes.byref(d)) == -1
        assert L.equigspr_attention_backward_work_size(ctypes.byref(d)) == -1
        assert L.equigspr_attention_forward(ctypes.byref(d), 16, None, None, None, None) == -2
    assert L.equigspr_attention_backward(ctypes.byref(_attention()), 16, None, 16, ctypes.byref(far), 16, None, None, None, None) == -2


def _splits(dtype, dim, nq, nk, batch=1, kv_heads=1, group=1):
    """Parts of the key axis, from the size of the workspace: a log-sum per row and part, rounded up to four, and a row of dim values."""
    d = _attention(dtype=dtype, dim=dim, nq=nq, nk=nk, batch=batch, heads=kv_heads * group, kv_heads=kv_heads)
    size, rows = _lib.lib().equigspr_attention_work_size(ctypes.byref(d)), batch * kv_heads * nq * group
    parts = [p for p in range(2, 2000) if (p * rows + 3) // 4 * 4 + p * rows * dim == size]
    return parts[0] if size else 1


@pytest.mark.parametrize("dtype,dim,tile", [(0, 8, 64), (0, 32, 64), (0, 33, 32), (0, 128, 32), (1, 8, 64), (2, 128, 64)])
def test_attention_key_axis_is_cut_once_for_every_four_tiles_at_most(dtype, dim, tile):
    for nk in (1, 4 * tile - 1, 4 * tile, 4 * tile + 1, 8 * tile - 1, 8 * tile, 1000, 3777, 16384):
        p = _splits(dtype, dim, 1, nk)
        assert p <= -(-nk // (4 * tile)), (nk, p)
    assert _splits(dtype, dim, 1, 16384) > 16                              # and there are many where a row is alone
