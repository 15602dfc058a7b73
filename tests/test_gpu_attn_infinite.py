"""GPU: infinities and the types' largest values in keys and values that are
attended. A product's operands enter it in two parts, and a part of an infinity
must not make a NaN of what IEEE arithmetic calls infinite, zero or finite.
Tolerances as derived in test_gpu_attn.py (`attn_reference`)."""
import math

import pytest

import moe_cuda as mc
import test_gpu_attn as ta

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
INF = math.inf
TYPES = [torch.bfloat16, torch.float16, torch.float32]
# one cluster, and pieces dealt to the whole GPU with a second launch
LENGTHS = [100, 3000]
SHAPES = [(4, 2, 64, 16), (16, 1, 128, 24), (7, 1, 256, 16), (2, 2, 80, 1)]


def put(c, table, s, t, val):
    ps = c.shape[1]
    c[int(table[s, t // ps]), t % ps] = val


def gathered(c, table, s, n, group):
    t = torch.arange(n, device="cuda")
    return c[table[s].long()[t // c.shape[1]], t % c.shape[1]].double().repeat_interleave(group, 1)


def case(dt, shape, n):
    n_q, n_kv, hd, ps = shape
    q, k, v, table = ta.make_attn(dt, 3, n_q, n_kv, hd, ps, [n, n, n], seed=n + hd)
    pos = torch.full((3,), n - 1, dtype=torch.int32, device="cuda")
    return q, k, v, table, pos, hd**-0.5


def rest_is_right(dt, args, out, lse, skip):
    """Every element outside `skip` [rows][n_q][hd] against the finite reference `args`."""
    q, k, v, table, pos, scale = args
    ta._sixteen[0] = dt != torch.float32
    ref, ref_lse, bound, lse_bound = ta.attn_reference(q, k, v, table, pos, range(3), scale)
    tiny = 2.0**-25 if dt == torch.float16 else 0.0
    err = (out.double() - ref).abs() - (bound + ta.u(dt) * (ref.abs() + bound) + tiny)
    assert (err[~skip] <= 0).all(), float(err[~skip].max())
    assert ((lse.double() - ref_lse).abs() <= lse_bound).all()


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("n", LENGTHS)
def test_infinite_values_make_infinite_outputs(gpu, dt, shape, n):
    """+inf, -inf and both at once in columns of one row's values: inf, -inf and
    NaN there, and nothing else changes. The weight is about that of any other
    position, so that it does not underflow."""
    q, k, v, table, pos, scale = case(dt, shape, n)
    group = shape[0] // shape[1]
    want_v = v.clone()
    for col, t, val in ((1, 37, INF), (2, 5, -INF), (3, n - 1, INF), (3, n // 2, -INF)):
        x = v[int(table[1, t // shape[3]]), t % shape[3]]
        x[0, col] = val
        want_v[int(table[1, t // shape[3]]), t % shape[3], 0, col] = 0
    out, lse = ta.run_attn(q, k, v, table, pos, scale, n)
    torch.cuda.synchronize()
    first = out[1, :group]
    assert (first[:, 1] == INF).all() and (first[:, 2] == -INF).all() and first[:, 3].isnan().all()
    skip = torch.zeros(out.shape, dtype=torch.bool, device="cuda")
    skip[1, :group, 1:4] = True
    rest_is_right(dt, (q, k, want_v, table, pos, scale), out, lse, skip)


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("n", LENGTHS)
def test_keys_of_minus_infinity_weigh_nothing(gpu, dt, shape, n):
    """Scores of -inf for a few positions of a row, and for all of another's;
    +inf makes a row NaN, and only its own key-value head."""
    q, k, v, table, pos, scale = case(dt, shape, n)
    q = q.abs() + 0.5
    out_of = [0, 17, n // 2, n - 1]
    for t in out_of:
        k[int(table[0, t // shape[3]]), t % shape[3], :, 3] = -INF
    for t in range(n):
        k[int(table[1, t // shape[3]]), t % shape[3], :, 5] = -INF
    k[int(table[2, 7 // shape[3]]), 7 % shape[3], 0, 6] = INF
    out, lse = ta.run_attn(q, k, v, table, pos, scale, n)
    torch.cuda.synchronize()
    group = shape[0] // shape[1]
    assert (out[1] == 0).all() and (lse[1] == -INF).all()
    assert out[2, :group].isnan().all() and not out[2, group:].isnan().any()
    kk, vv = gathered(k, table, 0, n, group), gathered(v, table, 0, n, group)
    live = torch.ones(n, dtype=torch.bool, device="cuda")
    live[out_of] = False
    x = torch.einsum("hd,nhd->hn", q[0].double(), kk[live]) * scale
    p = torch.softmax(x, 1)
    want = torch.einsum("hn,nhd->hd", p, vv[live])
    # the bounds of test_gpu_attn.py over the positions that count
    mag = (torch.einsum("hd,nhd->hn", q[0].double(), kk[live].abs()) * scale).amax(1)
    weight = (shape[2] + 8) * 2.0**-23 * mag + 2.0**-21 * mag + 2.0**-22 * (x.amax(1) - x.amin(1)) + 2.0**-20
    rel = 2 * weight + (2.0**-16 if dt != torch.float32 else 0) + (n / 16 + 200) * 2.0**-23
    bound = rel[:, None] * torch.einsum("hn,nhd->hd", p, vv[live].abs())
    tiny = 2.0**-25 if dt == torch.float16 else 0.0
    assert ((out[0].double() - want).abs() <= bound + ta.u(dt) * (want.abs() + bound) + tiny).all()
    ref_lse = torch.logsumexp(x, 1)
    assert ((lse[0].double() - ref_lse).abs() <= weight + (n / 16 + 200) * 2.0**-23 + 2.0**-22 * ref_lse.abs()).all()


@pytest.mark.parametrize("n", LENGTHS)
def test_the_largest_fp32_numbers(gpu, n):
    """fp32 numbers next to the largest, which no 11-bit part holds: a value
    of that size has a finite share, and a key's meets a query's zero."""
    q, k, v, table, pos, scale = case(torch.float32, (4, 2, 64, 16), n)
    big = torch.finfo(torch.float32).max
    q[:, :, 9] = 0
    for t in (3, n - 2):
        k[int(table[0, t // 16]), t % 16, :, 9] = big
        v[int(table[2, t // 16]), t % 16, 1, 4] = big / 2 if t == 3 else -big
    out, lse = ta.run_attn(q, k, v, table, pos, scale, n)
    torch.cuda.synchronize()
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    rest_is_right(torch.float32, (q, k, v, table, pos, scale), out, lse, torch.zeros(out.shape, dtype=torch.bool, device="cuda"))


@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_an_empty_row_is_zero_whatever_its_values_hold(gpu, dt):
    """Every score -inf: zeros, also over infinite and NaN values."""
    q, k, v, table, pos, scale = case(dt, (4, 2, 64, 16), 100)
    q = q.abs() + 0.5
    for t in range(100):
        k[int(table[1, t // 16]), t % 16, :, 5] = -INF
    v[int(table[1, 2]), 3, :, 7] = INF
    v[int(table[1, 4]), 4, :, 8] = math.nan
    out, lse = ta.run_attn(q, k, v, table, pos, scale, 100)
    torch.cuda.synchronize()
    assert (out[1] == 0).all() and (lse[1] == -INF).all() and torch.isfinite(out[0]).all() and torch.isfinite(out[2]).all()
