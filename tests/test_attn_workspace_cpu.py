"""CPU: the workspace of attention calls of many rows. Rows that fill the GPU by
themselves need no share of it each for every stretch of a long context."""
import ctypes as C

import pytest

import moe_cuda as mc

P = 0x7000_0000_0000


def size(rows, n_q, hd, max_kv, n_kv=4):
    c = mc.MoeKvCache(P, P, mc.BF16, 1 << 16, 16, n_kv, hd, 16 * n_kv * hd, n_kv * hd, hd)
    return mc.lib().moe_paged_attention_workspace(rows, n_q, C.byref(c), max_kv)


@pytest.mark.parametrize("rows,max_kv,most", [
    (32 * 4096, 4096, 100e6), (32 * 8192, 8192, 100e6),       # prompts of 32 sequences
    (8192, 8192, 300e6), (4096, 131072, 300e6), (1 << 20, 1 << 20, 100e6), (513, 1 << 20, 300e6)])
def test_many_rows_are_bounded(rows, max_kv, most):
    """32 query heads of 128: before this bound 17 and 70 GB for the first two."""
    assert size(rows, 32, 128, max_kv) <= most


def test_larger_contexts_never_need_less():
    for rows in (1, 32, 512, 513, 2000, 16384, 16385):
        need = [size(rows, 32, 128, kv) for kv in (1, 64, 2048, 2049, 4096, 8192, 20000, 131072, 1 << 20, 2**31 - 1)]
        assert need == sorted(need)


def test_few_hundred_rows_keep_a_part_for_512_positions():
    for rows, kv in ((513, 8192), (600, 5000), (1024, 8192)):
        assert size(rows, 4, 64, kv) == -(-kv // 512) * rows * 4 * 66 * 4 + 16
