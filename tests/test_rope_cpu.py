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


@pytest.mark.parametrize("over", [dict(k=P), dict(v=P + 64), dict(k=P + 3 * 512), dict(k=P + 128, ldk=256),
                                  dict(ldq=512, ldo=512, k=P + 512 - 128, ldk=512)])
def test_queries_in_place_over_keys_or_values_are_refused(over):
    """q_out = q: rows of 512 bytes that keys or values (256 bytes) lie in would be read after they were written."""
    d = dict(out=P, k=P + (1 << 20), v=P + (1 << 21))
    d.update(over)
    assert rope(**d) == INVALID and b"overlaps k or v" in mc.lib().moe_cuda_last_error()


def test_columns_of_one_projection_are_not_refused():
    """q, k and v beside one another, queries in place: it gets as far as the device."""
    rc = rope(ldq=512, ldo=512, out=P, k=P + 512, ldk=512, v=P + 768, ldv=512)
    assert rc not in (mc.MOE_ERR_INVALID, mc.MOE_ERR_UNSUPPORTED) or b"device memory" in mc.lib().moe_cuda_last_error()
