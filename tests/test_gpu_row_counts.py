"""GPU: row counts next to 2^31."""
import pytest

import moe_cuda as mc

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
ROWS = 2**31 - 1


def test_routing(gpu):
    """One expert, a few NaN logits among them: the lists of the first and the last rows, and of a row past 2^30."""
    x = torch.zeros(ROWS, 1, dtype=torch.bfloat16, device="cuda")
    nan = [0, 7, (1 << 30) + 5, ROWS - 1]
    x[nan] = float("nan")
    idx = torch.full((ROWS, 1), 5, dtype=torch.int32, device="cuda")
    p = torch.full((ROWS, 1), 5.0, device="cuda")
    mc.route(x, idx, p)
    torch.cuda.synchronize()
    for r in (0, 1, 7, 8, 1 << 30, (1 << 30) + 5, ROWS - 2, ROWS - 1):
        assert int(idx[r]) == (-1 if r in nan else 0) and float(p[r]) == (0 if r in nan else 1)
    assert int((idx == -1).sum()) == len(nan) and int((idx == 0).sum()) == ROWS - len(nan)
    del x, idx, p
    torch.cuda.empty_cache()
