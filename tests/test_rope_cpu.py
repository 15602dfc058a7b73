"""CPU: norm + rotation + append without rows, and queries in place across keys
or values. Arguments are checked before any CUDA call."""
import pytest

import moe_cuda as mc
from test_attn_cpu import INVALID, P, rope


def test_a_call_without_rows_needs_no_pointers():
    """As empty tensors give them."""
    assert rope(rows=0, q=None, out=None, k=None, v=None, pos=None, slot=None) == mc.MOE_OK
    assert rope(rows=0, n_q=0, q=None, out=None, k=None, v=None, pos=None, slot=P) == mc.MOE_OK
    assert rope(rows=0, q=None, out=None, pos=None, rot=12) == mc.MOE_ERR_UNSUPPORTED     # sizes are still checked
