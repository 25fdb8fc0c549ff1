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
