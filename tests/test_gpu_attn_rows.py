"""GPU: attention of very many rows, whose contexts are split less the more rows
there are; a sample of them against the 64-bit form of test_gpu_attn.py."""
import numpy as np
import pytest

import moe_cuda as mc
import test_gpu_attn as ta

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("dt", ta.TYPES, ids=str)
@pytest.mark.parametrize("rows,lens", [(2100, [2100, 9000, 40]), (16500, [16384, 3000, 116])])
def test_prompts_of_many_rows(gpu, dt, rows, lens):
    """Rows of three sequences, with padding among them; 7 parts a row and one."""
    q, k, v, table = ta.make_attn(dt, rows, 4, 2, 64, 16, lens, seed=rows)
    rng = np.random.default_rng(rows)
    seq = rng.integers(-1, 3, rows)
    pos = np.array([rng.integers(-1, lens[s]) if s >= 0 else 5 for s in seq])
    seq[:3], pos[:3] = (0, 1, 2), [n - 1 for n in lens]
    i32 = dict(dtype=torch.int32, device="cuda")
    sq, ps = torch.tensor(seq, **i32), torch.tensor(pos, **i32)
    out, lse = ta.run_attn(q, k, v, table, ps, 0.125, max(lens), sq)
    torch.cuda.synchronize()
    assert (out[sq < 0] == 7).all() and not out.isnan().any()
    some = torch.tensor([0, 1, 2, *rng.integers(3, rows, 40)], device="cuda")
    ta._sixteen[0] = dt != torch.float32
    ref, ref_lse, bound, lse_bound = ta.attn_reference(q[some], k, v, table, ps[some], sq[some], 0.125)
    tiny = 2.0**-25 if dt == torch.float16 else 0.0
    err = (out[some].double() - ref).abs() - (bound + ta.u(dt) * (ref.abs() + bound) + tiny)
    live = sq[some] >= 0
    assert (err[live] <= 0).all()
    full = live & (ps[some] >= 0)
    assert ((lse[some].double() - ref_lse).abs()[full] <= lse_bound[full]).all()
