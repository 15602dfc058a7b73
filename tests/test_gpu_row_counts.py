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


def test_append(gpu):
    """Rows without a slot but for four, all with the same keys and values."""
    k = torch.arange(1, 9, device="cuda").bfloat16().view(1, 1, 8).expand(ROWS, 1, 8)
    kc, vc = (torch.zeros(4, 4, 1, 8, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    slot = torch.full((ROWS,), -1, dtype=torch.int32, device="cuda")
    for r, s in ((0, 3), ((1 << 30) + 1, 9), (ROWS - 2, 0), (ROWS - 1, 15)):
        slot[r] = s
    mc.qk_norm_rope(None, k, k, kc, vc, None, slot, None)
    torch.cuda.synchronize()
    want = torch.zeros(16, 8, dtype=torch.bfloat16, device="cuda")
    want[[3, 9, 0, 15]] = k[0, 0]
    assert torch.equal(kc.view(16, 8), want) and torch.equal(vc.view(16, 8), want)
    del slot
    torch.cuda.empty_cache()
