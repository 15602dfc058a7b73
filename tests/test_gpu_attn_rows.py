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


@pytest.mark.parametrize("rows", [64, 8300])
def test_long_sums_are_not_cut(gpu, rows):
    """131072 positions of positive values, split over the GPU and (rows beyond
    8192) in one part, 2048 steps a warp: the mean signed error of 65536 outputs.
    An f16 rounding is off by up to 2^-11, either way: 2^-11 / sqrt(3) / 256 = 1.1e-6
    of their mean, five times that 6e-6. A step's sum loses at most 2^-22 by the tensor
    core's truncation, an fp32 addition as much either way. Errors of the scores
    move weights between values that do not depend on the keys: as often up as
    down. 2e-5 leaves room for three times all of it; sums kept in the tensor
    core throughout lose 2.3e-4."""
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    n, hd, ps, nq = 131072, 128, 64, 8
    k = torch.randn(n // ps, ps, 1, hd, generator=g, device="cuda").half()
    v = (torch.randn(n // ps, ps, 1, hd, generator=g, device="cuda").abs() + 0.5).half()
    table = torch.randperm(n // ps, generator=g, device="cuda").int()[None]
    some = (1.5 * torch.randn(64, nq, hd, generator=g, device="cuda")).half()
    q = some.repeat(-(-rows // 64), 1, 1)[:rows].contiguous()
    i32 = dict(dtype=torch.int32, device="cuda")
    out, _ = ta.run_attn(q, k, v, table, torch.full((rows,), n - 1, **i32), hd**-0.5, n, torch.zeros(rows, **i32))
    kk, vv = (c[table[0].long()].reshape(n, hd).double() for c in (k, v))
    want = (torch.softmax(some.double().reshape(-1, hd) @ kk.T * hd**-0.5, 1) @ vv).reshape(64, nq, hd)
    assert abs(float((out[:64].double() - want).sum() / want.sum())) < 2e-5
