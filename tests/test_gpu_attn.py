"""GPU: planning, norm + rotation + append, and attention over a paged cache,
against plain 64-bit forms, at the sizes, layouts and masks where they can go
wrong; and the three together with expert routing and the MoE block, captured
into one graph and replayed.

Tolerances. u(t) = finfo(t).eps / 2 is the rounding of a stored result. The
fp32 work before it is bounded by operation counts, each operation at most
2^-24 (2^-23 inside the tensor core, whose sums truncate), as derived at
`attn_bound` and `rope_bound`."""
import math

import numpy as np
import pytest

import moe_cuda as mc

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

NAN = float("nan")


def u(dt):
    return torch.finfo(dt).eps / 2


# ---- attention -----------------------------------------------------------------

def attn_reference(q, k, v, table, pos, row_seq, scale):
    """(out, lse, bound) in 64 bits, row by row; keys on pages outside the
    cache or past the table are not attended. bound is what the kernel's fp32
    work may be off before the result is stored."""
    q, k, v = q.double(), k.double(), v.double()
    R, nq, hd = q.shape
    n_pages, ps, nkv, _ = k.shape
    mp = table.shape[1]
    out = torch.zeros_like(q)
    lse = torch.full((R, nq), -math.inf, dtype=torch.float64, device=q.device)
    bound, lse_bound = torch.zeros_like(q), torch.zeros_like(lse)
    for r in range(R):
        s = int(row_seq[r])
        if not 0 <= s < table.shape[0]:
            continue
        n = min(int(pos[r]) + 1, mp * ps)
        t = torch.arange(max(n, 0), device=q.device)
        page = table[s].long()[t // ps]
        t, page = t[(page >= 0) & (page < n_pages)], page[(page >= 0) & (page < n_pages)]
        if len(t) == 0:
            continue
        kk = k[page, t % ps].repeat_interleave(nq // nkv, 1)          # [n, nq, hd]
        vv = v[page, t % ps].repeat_interleave(nq // nkv, 1)
        x = torch.einsum("hd,nhd->hn", q[r], kk) * scale
        lse[r] = torch.logsumexp(x, 1)
        p = torch.exp(x - lse[r][:, None])
        out[r] = torch.einsum("hn,nhd->hd", p, vv)
        # a score: hd products and sums (the fp32 path splits each product in
        # three and drops 2^-22 of it), the scale, log2 e and the reference's
        # subtraction; a weight: that absolute error of its exponent, exp2 and
        # its split into two 16-bit numbers (2^-16; fp32: 2^-21)
        mag = (torch.einsum("hd,nhd->hn", q[r].abs(), kk.abs()) * abs(scale)).amax(1)
        score = (hd + 8) * 2.0**-23 * mag + 2.0**-21 * mag + 2.0**-22 * (x.amax(1) - x.amin(1))
        weight = score + 2.0**-20
        # numerator and sum both carry the weights' errors; len/16 steps and up
        # to 200 joins add to them
        rel = 2 * weight + 2.0**-16 * (k_type_16(q)) + (len(t) / 16 + 200) * 2.0**-23
        bound[r] = rel[:, None] * torch.einsum("hn,nhd->hd", p, vv.abs())
        lse_bound[r] = weight + (len(t) / 16 + 200) * 2.0**-23 + 2.0**-22 * lse[r].abs()
    return out, lse, bound, lse_bound


_sixteen = [True]


def k_type_16(_):
    return 1.0 if _sixteen[0] else 0.0


def make_attn(dt, rows, n_q, n_kv, hd, ps, lens, seed=0, spare=2, layout="nphd", row_seq=None, mp=None):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    lens = list(lens)
    n_seq = len(lens)
    mp = mp or max(1, max(-(-max(n, 1) // ps) for n in lens))
    n_pages = sum(-(-max(n, 0) // ps) for n in lens) + spare
    shape = (n_pages, ps, n_kv, hd)
    if layout == "nphd":
        k, v = torch.full(shape, NAN, device="cuda", dtype=dt), torch.full(shape, NAN, device="cuda", dtype=dt)
    else:                                              # heads outside the tokens of a page
        k, v = (torch.full((n_pages, n_kv, ps, hd), NAN, device="cuda", dtype=dt).transpose(1, 2) for _ in range(2))
    order = torch.randperm(n_pages, generator=g, device="cuda").tolist()
    table = torch.full((n_seq, mp), 2**30, dtype=torch.int32, device="cuda")      # entries past the end are junk
    for s, n in enumerate(lens):
        for j in range(-(-max(n, 0) // ps)):
            page = order.pop()
            if j < mp:
                table[s, j] = page
            m = min(ps, n - j * ps)
            k[page, :m] = torch.randn(m, n_kv, hd, generator=g, device="cuda").to(dt)
            v[page, :m] = torch.randn(m, n_kv, hd, generator=g, device="cuda").to(dt)
    q = (1.5 * torch.randn(rows, n_q, hd, generator=g, device="cuda")).to(dt)
    return q, k, v, table


def run_attn(q, k, v, table, pos, scale, max_kv, row_seq=None, out=None, stream=None, lse=True):
    R, nq, hd = q.shape
    out = torch.full((R, nq, hd), 7.0, device="cuda", dtype=k.dtype) if out is None else out
    ls = torch.full((R, nq), 7.0, device="cuda") if lse else None
    n = mc.paged_attention_workspace(R, nq, k, v, max_kv)
    ws = torch.full((max(n, 1),), 255, dtype=torch.uint8, device="cuda")         # every float a NaN
    mc.paged_attention(q, k, v, table, pos, out, ws if n else None, max_kv, scale, lse=ls, row_seq=row_seq, stream=stream)
    return out, ls


def check_attn(q, k, v, table, pos, row_seq=None, max_kv=None, scale=None):
    scale = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    pos = torch.tensor(pos, dtype=torch.int32, device="cuda")
    rs = None if row_seq is None else torch.tensor(row_seq, dtype=torch.int32, device="cuda")
    max_kv = max_kv or table.shape[1] * k.shape[1]
    out, lse = run_attn(q, k, v, table, pos, scale, max_kv, rs)
    torch.cuda.synchronize()
    _sixteen[0] = q.dtype != torch.float32
    ref, ref_lse, bound, lse_bound = attn_reference(q, k, v, table, pos, range(len(pos)) if rs is None else rs, scale)
    live = [r for r in range(len(pos)) if rs is None or 0 <= int(rs[r]) < table.shape[0]]
    dead = [r for r in range(len(pos)) if r not in live]
    assert (out[dead] == 7).all() and (lse[dead] == 7).all()
    tiny = 2.0**-25 if q.dtype == torch.float16 else 0.0
    err = (out.double() - ref).abs() - (bound + u(q.dtype) * (ref.abs() + bound) + tiny)
    assert not out[live].isnan().any()
    assert (err[live] <= 0).all(), float(err[live].max())
    fin = torch.isfinite(ref_lse)
    keep = torch.zeros_like(fin)
    keep[live] = True
    assert torch.equal(lse.double()[keep & ~fin], ref_lse[keep & ~fin])
    el = (lse.double() - ref_lse).abs()[keep & fin] - lse_bound[keep & fin]
    assert (el <= 0).all(), float(el.max())
    return out, lse


TYPES = [torch.bfloat16, torch.float16, torch.float32]
EDGES = [0, 1, 2, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 500]


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("n_q,n_kv,hd,ps", [(32, 4, 128, 16), (8, 8, 64, 16), (16, 1, 128, 64), (9, 1, 80, 5),
                                            (40, 2, 96, 1), (4, 2, 16, 16), (7, 1, 256, 24), (32, 1, 256, 16),
                                            (6, 3, 8, 3), (5, 5, 200, 128), (64, 2, 64, 33)])
def test_attention_at_edge_lengths(gpu, dt, n_q, n_kv, hd, ps):
    q, k, v, table = make_attn(dt, len(EDGES), n_q, n_kv, hd, ps, EDGES, seed=n_q + hd)
    check_attn(q, k, v, table, [n - 1 for n in EDGES])


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("n", [1, 511, 4097, 20011])
def test_attention_of_one_row(gpu, dt, n):
    """One row split over the GPU: from a single run to the largest number of them."""
    q, k, v, table = make_attn(dt, 1, 8, 1, 128, 16, [n], seed=n)
    check_attn(q, k, v, table, [n - 1])


@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_attention_hint_too_small_or_large(gpu, dt):
    """max_kv only sets the split: any value gives the same attention."""
    lens = [900, 3, 2050]
    q, k, v, table = make_attn(dt, 3, 8, 2, 64, 16, lens, seed=5)
    for hint in (1, 64, 700, 100000, 2**31 - 1):
        check_attn(q, k, v, table, [n - 1 for n in lens], max_kv=hint)


@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_attention_rows_of_one_sequence_and_padding(gpu, dt):
    """Rows name their sequence: several new tokens of one, out of order, and padding that stays as it was."""
    lens = [70, 200, 1]
    q, k, v, table = make_attn(dt, 8, 12, 3, 64, 16, lens, seed=6)
    check_attn(q, k, v, table, [199, 69, 198, 0, 5, 150, -1, 0], row_seq=[1, 0, 1, 2, -1, 1, 0, 3])


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("ps", [16, 24])
def test_attention_layout_strides_and_bad_pages(gpu, dt, ps):
    """Heads outside tokens in a page; q and out as slices of wider rows; pages
    outside the cache (their keys are not attended, even all of them);
    a position past the table."""
    lens = [300, 77, 40]
    q, k, v, table = make_attn(dt, 3, 8, 2, 128, ps, lens, seed=7, layout="nhpd")
    wide = torch.full((3, 1280), NAN, device="cuda", dtype=dt)
    wide[:, 128:1152] = q.flatten(1)
    q = wide[:, 128:1152].unflatten(1, (8, 128))
    table[0, 2], table[0, 5] = -1, k.shape[0]
    table[1, :] = 2**31 - 1
    check_attn(q, k, v, table, [299, 76, 39])
    q2, k2, v2, t2 = make_attn(dt, 1, 4, 2, 64, ps, [5 * ps], seed=8, mp=3)
    check_attn(q2, k2, v2, t2, [5 * ps - 1])
    out = torch.full((3, 1280), 3.0, device="cuda", dtype=dt)
    pos = torch.tensor([299, 76, 39], dtype=torch.int32, device="cuda")
    run_attn(q, k, v, table, pos, 0.1, 300, out=out[:, 128:1152].unflatten(1, (8, 128)))
    ref, _ = run_attn(q, k, v, table, pos, 0.1, 300)
    assert torch.equal(out[:, 128:1152], ref.flatten(1)) and (out[:, :128] == 3).all() and (out[:, 1152:] == 3).all()


@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_attention_scores_far_apart(gpu, dt):
    """Scores that rise along the row by far more than the reference may lag,
    a dominating first key, scores all alike, and large negative ones."""
    n, hd = 700, 64
    q, k, v, table = make_attn(dt, 4, 2, 1, hd, 16, [n] * 4, seed=9)
    q[:] = 0
    q[:, :, 0] = 1
    ramp = torch.linspace(0, 200, n, device="cuda")
    for s, x in enumerate((ramp, ramp.flip(0), torch.zeros(n, device="cuda"), -ramp - 300)):
        page = table[s].long()[torch.arange(n, device="cuda") // 16]
        k[page, torch.arange(n, device="cuda") % 16, 0, 0] = x.to(dt)
    check_attn(q, k, v, table, [n - 1] * 4, scale=1.0)


@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_attention_nonfinite_keys_attended(gpu, dt):
    """A NaN key that is attended makes its row NaN, and only that row and its
    key-value head; -inf scores weigh nothing; all of them -inf is an empty row."""
    q, k, v, table = make_attn(dt, 3, 4, 2, 64, 16, [100, 100, 100], seed=10)
    q = q.abs()
    k[int(table[0, 3]), 5, 1, 0] = NAN
    pos = torch.full((3,), 99, dtype=torch.int32, device="cuda")
    if dt != torch.float32:                       # an infinite fp32 key splits into inf and NaN parts: not finite either way
        k[int(table[1, 0]), 2, :, 3] = -math.inf
        for t in range(100):
            k[int(table[2, t // 16]), t % 16, :, 3] = -math.inf
    out, lse = run_attn(q, k, v, table, pos, 0.125, 100)
    assert out[0, 2:].isnan().all() and lse[0, 2:].isnan().all() and not out[0, :2].isnan().any()
    if dt != torch.float32:
        k[int(table[1, 0]), 2] = 0
        k2, v2 = k.clone(), v.clone()
        ref = attn_reference(q[1:2], k2, v2, table[1:2], pos[1:2], [0], 0.125)
        w = math.e**0                            # the key with a -inf score is left out of the sum: compare without it
        x = torch.einsum("hd,nhd->hn", q[1].double(), k2[table[1].long()[torch.arange(100, device="cuda") // 16],
                                                        torch.arange(100, device="cuda") % 16].double().repeat_interleave(2, 1)) * 0.125
        x[:, 2] = -math.inf
        p = torch.softmax(x, 1)
        vv = v2[table[1].long()[torch.arange(100, device="cuda") // 16], torch.arange(100, device="cuda") % 16].double().repeat_interleave(2, 1)
        want = torch.einsum("hn,nhd->hd", p, vv)
        _sixteen[0] = True
        assert ((out[1].double() - want).abs() <= 2 * ref[2][0] + u(dt) * want.abs() + 2.0**-25).all() and w == 1
        assert (out[2] == 0).all() and (lse[2] == -math.inf).all()


def test_attention_offsets_past_32_bits(gpu):
    """Pages so far apart that element offsets pass 2^32."""
    ps, nkv, hd, far = 16, 2, 64, (1 << 31) + 4096
    buf = torch.empty(2 * far + 2 * ps * nkv * hd, dtype=torch.bfloat16, device="cuda")
    half = ps * nkv * hd
    k = buf.as_strided((3, ps, nkv, hd), (far, nkv * hd, hd, 1), 0)
    v = buf.as_strided((3, ps, nkv, hd), (far, nkv * hd, hd, 1), half)
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    for p in range(3):
        k[p] = torch.randn(ps, nkv, hd, generator=g, device="cuda").bfloat16()
        v[p] = torch.randn(ps, nkv, hd, generator=g, device="cuda").bfloat16()
    table = torch.tensor([[2, 0, 1], [1, 2, 0]], dtype=torch.int32, device="cuda")
    q = torch.randn(2, 4, hd, generator=g, device="cuda").bfloat16()
    check_attn(q, k, v, table, [44, 17])
    # and the append into the farthest page
    new = torch.randn(1, nkv, hd, generator=g, device="cuda").bfloat16()
    slot = torch.tensor([2 * ps + 7], dtype=torch.int32, device="cuda")
    mc.qk_norm_rope(None, new, new, k, v, None, slot, None)
    assert torch.equal(k[2, 7], new[0]) and torch.equal(v[2, 7], new[0])


def test_attention_in_place_repeatable_and_on_another_stream(gpu):
    """out may be q; the same call gives the same bits, with any contents of
    the workspace, also on two streams at once with a workspace each."""
    lens = [3000, 1, 900, 64]
    q, k, v, table = make_attn(torch.bfloat16, 4, 8, 2, 128, 16, lens, seed=11)
    pos = torch.tensor([n - 1 for n in lens], dtype=torch.int32, device="cuda")
    ref, ref_lse = run_attn(q, k, v, table, pos, 0.09, 3000)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(8):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(run_attn(q, k, v, table, pos, 0.09, 3000, stream=s))
    torch.cuda.synchronize()
    for o, l in got:
        assert torch.equal(o, ref) and torch.equal(l, ref_lse)
    q2 = q.clone()
    run_attn(q2, k, v, table, pos, 0.09, 3000, out=q2)
    torch.cuda.synchronize()
    assert torch.equal(q2, ref)


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("hint", [64, 2048, 6000])
def test_attention_of_many_rows(gpu, dt, hint):
    """More rows than are dealt evenly, of a few sequences of very different
    lengths, with padding among them; the hint picks one CTA a row, or runs."""
    lens = [5000, 1, 130, 2300]
    q, k, v, table = make_attn(dt, 700, 4, 2, 64, 16, lens, seed=12)
    rng = np.random.default_rng(2)
    seq = rng.integers(-1, 4, 700)
    pos = [int(rng.integers(-1, lens[s])) if s >= 0 else 3 for s in seq]
    pos[5], seq[5] = 4999, 0
    check_attn(q, k, v, table, pos, row_seq=seq.tolist(), max_kv=hint)


def test_calls_that_follow_one_another_on_one_workspace(gpu):
    """Calls of different sizes and types, each of which leaves its partial
    results in the same workspace, with nothing waiting between them."""
    sets = []
    for i, (dt, rows, n_q, n_kv, hd, lens) in enumerate([
            (torch.bfloat16, 3, 8, 2, 128, [4000, 100, 2500]), (torch.float16, 1, 16, 1, 64, [9000]),
            (torch.float32, 2, 4, 4, 128, [3000, 70]), (torch.bfloat16, 2, 32, 1, 256, [2100, 2200])]):
        q, k, v, table = make_attn(dt, rows, n_q, n_kv, hd, 16, lens, seed=20 + i)
        pos = torch.tensor([n - 1 for n in lens], dtype=torch.int32, device="cuda")
        sets.append((q, k, v, table, pos, max(lens)))
    alone = []
    for q, k, v, table, pos, most in sets:
        alone.append(run_attn(q, k, v, table, pos, 0.1, most)[0])
        torch.cuda.synchronize()
    need = max(mc.paged_attention_workspace(s[0].shape[0], s[0].shape[1], s[1], s[2], s[5]) for s in sets)
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    outs = []
    for _ in range(5):
        for q, k, v, table, pos, most in sets:
            out = torch.empty_like(q)
            mc.paged_attention(q, k, v, table, pos, out, ws, most, 0.1)
            outs.append(out)
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        assert torch.equal(out, alone[i % len(sets)])


def test_a_step_written_just_before_it_is_read(gpu):
    """Planning, append and attention follow one another on one stream over and
    over with nothing in between: each sees what the one before it wrote."""
    n_seq, nkv, hd, ps, n_pages = 7, 2, 64, 4, 400
    i32 = dict(dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda")
    g.manual_seed(8)
    steps = 60
    kv = torch.randn(steps, 2, n_seq, nkv, hd, generator=g, device="cuda").bfloat16()
    q = torch.randn(n_seq, 4, hd, generator=g, device="cuda").bfloat16()
    past, new, head = torch.zeros(n_seq, **i32), torch.ones(n_seq, **i32), torch.zeros(1, **i32)
    free, table, rows = torch.randperm(n_pages, generator=g, device="cuda").int(), torch.full((n_seq, 16), -1, **i32), torch.zeros(3, n_seq, **i32)
    kc, vc = (torch.zeros(n_pages, ps, nkv, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    outs = torch.zeros(steps, n_seq, 4, hd, dtype=torch.bfloat16, device="cuda")
    for t in range(steps):
        mc.kv_plan(past, new, ps, n_pages, free, table, rows[0], rows[1], rows[2], kv_len=past, free_head=head, free_head_out=head)
        mc.qk_norm_rope(None, kv[t, 0], kv[t, 1], kc, vc, rows[1], rows[2], None)
        mc.paged_attention(q, kc, vc, table, rows[1], outs[t], None, 64, 0.125, row_seq=rows[0])
    torch.cuda.synchronize()
    K = kv[:, 0].double().repeat_interleave(2, 2)                       # [steps, seq, 4, hd]
    V = kv[:, 1].double().repeat_interleave(2, 2)
    for t in range(steps):
        x = torch.einsum("shd,nshd->shn", q.double(), K[:t + 1]) * 0.125
        w = torch.softmax(x, 2)
        want = torch.einsum("shn,nshd->shd", w, V[:t + 1])
        # |x| < 2^4: fp32 scores within 2^-14, weights with their 2^-16
        assert near(outs[t], want, 2.0**-13 * torch.einsum("shn,nshd->shd", w, V[:t + 1].abs()))


# ---- norm, rotation and append ---------------------------------------------------

def rope_table(n, rot, theta=1e6):
    i = torch.arange(0, rot, 2, dtype=torch.float64)
    a = torch.arange(n, dtype=torch.float64)[:, None] * theta ** (-i / rot)
    return torch.cat([a.cos(), a.sin()], 1).float().cuda()


def rope_reference(x, w, eps, table, pos):
    """(result, bound), the bound in units of 2^-24 of the two numbers that make
    up a result: the sum of squares errs by at most hd (halved by the root),
    its mean and eps by 2 (halved), rsqrt by 2 ulp (4), the weight times the
    cosine or sine by 1, the product with x and the sum by 2, the product with
    rsqrt by 1, and the 64-bit form rounds the same table: hd/2 + 9, and 3 to
    spare for the halves' rounding up."""
    x, hd = x.double(), x.shape[-1]
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    mag = x.abs()
    rot = 0 if table is None else table.shape[1]
    if rot:
        c, s = table[pos.long()].double()[:, None, :].chunk(2, -1)
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat([a * c - b * s, b * c + a * s, x[..., rot:]], -1)
        both = mag[..., :rot // 2] + mag[..., rot // 2:rot]
        mag = torch.cat([both, both, mag[..., rot:]], -1)
    else:
        y = x
    return y, (hd / 2 + 12) * 2.0**-24 * mag * (1 if w is not None or rot else 0)


def near(got, want, bound):
    dt = got.dtype
    tiny = 2.0**-25 if dt == torch.float16 else 0.0
    err = (got.double() - want).abs() - (bound + u(dt) * (want.abs() + bound) + tiny)
    return bool((err <= 0).all())


@pytest.mark.parametrize("ti,to", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                   (torch.float32, torch.float32), (torch.float32, torch.bfloat16),
                                   (torch.float32, torch.float16)], ids=str)
@pytest.mark.parametrize("n_q,n_kv,hd,rot,ps,rows", [(32, 4, 128, 128, 16, 5), (4, 2, 16, 16, 16, 33), (7, 1, 80, 40, 5, 3),
                                                     (3, 3, 96, 96, 1, 2), (8, 2, 256, 64, 24, 7), (5, 1, 8, 8, 3, 1),
                                                     (2, 2, 200, 8, 16, 9), (40, 8, 128, 64, 16, 1300), (1, 1, 24, 16, 2, 4)])
@pytest.mark.parametrize("norm", [True, False])
def test_norm_rope_append(gpu, ti, to, n_q, n_kv, hd, rot, ps, rows, norm):
    g = torch.Generator(device="cuda")
    g.manual_seed(hd + rows)
    qkv = (3 * torch.randn(rows, (n_q + 2 * n_kv) * hd + 16, generator=g, device="cuda")).to(ti)
    q = qkv[:, :n_q * hd].unflatten(1, (n_q, hd))
    k = qkv[:, n_q * hd:(n_q + n_kv) * hd].unflatten(1, (n_kv, hd))
    v = qkv[:, (n_q + n_kv) * hd:(n_q + 2 * n_kv) * hd].unflatten(1, (n_kv, hd))
    n_pages = -(-rows // ps) + 3
    kc = torch.randn(n_pages, ps, n_kv, hd, generator=g, device="cuda").to(to)
    vc = torch.randn(n_pages, n_kv, ps, hd, generator=g, device="cuda").to(to).transpose(1, 2).contiguous()
    slot = torch.randperm(n_pages * ps, generator=g, device="cuda")[:rows].int()
    table = rope_table(50001, rot)
    pos = torch.randint(0, 50001, (rows,), generator=g, device="cuda", dtype=torch.int32)
    pos[0] = 50000
    if rows > 2:
        pos[1], pos[2], slot[-1] = -1, 50001, (n_pages * ps if rows > 4 else -1)
    w = [1 + 0.3 * torch.randn(hd, generator=g, device="cuda") if norm else None for _ in range(2)]
    out = torch.full((rows, n_q * hd + 8), 9.0, device="cuda", dtype=to)
    kc0, vc0 = kc.clone(), vc.clone()
    mc.qk_norm_rope(q, k, v, kc, vc, pos, slot, out[:, :n_q * hd].unflatten(1, (n_q, hd)), rope=table, q_norm=w[0],
                    k_norm=w[1], eps=1e-6)
    torch.cuda.synchronize()
    live = (pos >= 0) & (pos < 50001)
    got = out[:, :n_q * hd].unflatten(1, (n_q, hd))
    p = pos.clamp(0, 50000)
    assert near(got[live], *(x[live] for x in rope_reference(q, w[0], 1e-6, table, p)))
    assert (got[~live] == 9).all() and (out[:, n_q * hd:] == 9).all()
    put = live & (slot >= 0) & (slot < n_pages * ps)
    sl = slot[put].long()
    want_k, bound = rope_reference(k, w[1], 1e-6, table, p)
    assert near(kc[sl // ps, sl % ps], want_k[put], bound[put])
    assert torch.equal(vc[sl // ps, sl % ps], v[put].to(to))
    rest = torch.ones(n_pages * ps, dtype=torch.bool, device="cuda")
    rest[sl] = False
    assert torch.equal(kc.reshape(-1, n_kv, hd)[rest], kc0.reshape(-1, n_kv, hd)[rest])
    assert torch.equal(vc.reshape(-1, n_kv, hd)[rest], vc0.reshape(-1, n_kv, hd)[rest])
    # in place, queries only, keys and values only: the same bits
    if ti == to:
        q2 = qkv.clone()
        qi = q2[:, :n_q * hd].unflatten(1, (n_q, hd))
        mc.qk_norm_rope(qi, None, None, kc, vc, pos, None, qi, rope=table, q_norm=w[0], eps=1e-6)
        assert torch.equal(qi[live], got[live]) and torch.equal(q2[:, n_q * hd:], qkv[:, n_q * hd:])
        assert torch.equal(qi[~live], q[~live])
    k2, v2 = kc0.clone(), vc0.clone()
    mc.qk_norm_rope(None, k, v, k2, v2, pos, slot, None, rope=table, k_norm=w[1], eps=1e-6)
    assert torch.equal(k2, kc) and torch.equal(v2, vc)


def test_outputs_beside_their_inputs_in_one_matrix(gpu):
    """Inputs and outputs that are columns of one matrix do not overlap: the
    same bits as apart, and the other columns stay."""
    R, nq, nk, hd, ps = 7, 4, 2, 64, 16
    q, kc, vc, table = make_attn(torch.bfloat16, R, nq, nk, hd, ps, [40, 1, 5000, 64, 16, 700, 3], seed=21)
    pos = torch.tensor([39, 0, 4999, 63, 15, 699, 2], dtype=torch.int32, device="cuda")
    n, m = nq * hd, nk * hd
    x = torch.randn(R, n + 2 * m + 2 * n + 8, device="cuda").bfloat16()
    col = lambda t, a, h: t[:, a:a + h * hd].unflatten(1, (h, hd))
    ins = lambda t: (col(t, n, nq), col(t, 2 * n, nk), col(t, 2 * n + m, nk))      # q_out, q, k, v, attention's out
    rope = rope_table(5000, hd)
    slot = torch.arange(R, dtype=torch.int32, device="cuda")
    apart, kr, vr = torch.empty(R, nq, hd, device="cuda", dtype=torch.bfloat16), torch.zeros_like(kc), torch.zeros_like(vc)
    mc.qk_norm_rope(*ins(x), kr, vr, pos, slot, apart, rope=rope)
    y, k2, v2 = x.clone(), torch.zeros_like(kc), torch.zeros_like(vc)
    mc.qk_norm_rope(*ins(y), k2, v2, pos, slot, col(y, 0, nq), rope=rope)
    assert torch.equal(col(y, 0, nq), apart) and torch.equal(y[:, n:], x[:, n:])
    assert torch.equal(k2, kr) and torch.equal(v2, vr)
    want, _ = run_attn(apart, kc, vc, table, pos, 0.1, 5000)
    run_attn(col(y, 0, nq), kc, vc, table, pos, 0.1, 5000, out=col(y, 2 * n + 2 * m, nq))
    assert torch.equal(col(y, 2 * n + 2 * m, nq), want) and torch.equal(col(y, 0, nq), apart)
    assert torch.equal(y[:, n:2 * n + 2 * m], x[:, n:2 * n + 2 * m]) and torch.equal(y[:, -8:], x[:, -8:])


def test_append_without_rotation_copies(gpu):
    """rot_dim 0 and no norm: the rows arrive unchanged, whatever they hold."""
    kv = torch.tensor([NAN, math.inf, -math.inf, -0.0, 1e-40, 65504.0, 1.0, 2.0], device="cuda").repeat(6, 1, 1)
    kc, vc = torch.zeros(2, 4, 1, 8, device="cuda"), torch.zeros(2, 4, 1, 8, device="cuda")
    slot = torch.tensor([7, 0, 3, -1, 8, 5], dtype=torch.int32, device="cuda")
    mc.qk_norm_rope(None, kv, kv, kc, vc, None, slot, None)
    for s in range(8):
        want = kv[0, 0] if s in (7, 0, 3, 5) else torch.zeros(8, device="cuda")
        for c in (kc, vc):
            assert torch.equal(c.view(8, 8)[s].view(torch.int32), want.view(torch.int32))


# ---- planning -------------------------------------------------------------------

def plan_reference(past, new, ps, n_pages, free, head, table, cap):
    table = table.copy()
    mp = table.shape[1]
    head = min(max(head, 0), len(free))
    top, rows, asked, at = 2**31 - 1, [], 0, head
    kv = []
    for s in range(len(new)):
        p = max(int(past[s]), 0)
        n = min(max(int(new[s]), 0), top - p)
        held, need = min(-(-p // ps), mp), min(-(-(p + n) // ps), mp)
        for j in range(held, need):
            table[s, j] = free[at] if at < len(free) else -1
            at += 1
        asked += need - held
        kv.append(p + n)
        for t in range(p, p + min(n, cap + 1)):
            page = table[s, t // ps] if t // ps < mp else -1
            rows.append((s, t, page * ps + t % ps if 0 <= page < n_pages else -1))
    taken = min(asked, len(free) - head)
    total = min(sum(min(max(int(n), 0), top - max(int(p), 0)) for p, n in zip(past, new)), top)
    out = np.full((3, cap), -1, np.int32)
    for i, r in enumerate(rows[:cap]):
        out[:, i] = r
    return table, kv, out, head + taken, [total, asked, taken]


def run_plan(past, new, ps, n_pages, free, head, table, cap, alias=False):
    t = lambda x: torch.tensor(np.asarray(x, np.int32), device="cuda")  # noqa: E731
    past_d, new_d, free_d, head_d, table_d = t(past), t(new), t(free), t([head]), t(table)
    kv = past_d if alias else torch.empty_like(past_d)
    head_o = head_d if alias else torch.empty_like(head_d)
    rows, status = torch.full((3, cap), 5, dtype=torch.int32, device="cuda"), torch.empty(3, dtype=torch.int32, device="cuda")
    mc.kv_plan(past_d, new_d, ps, n_pages, free_d, table_d, rows[0], rows[1], rows[2], kv_len=kv, free_head=head_d,
               free_head_out=head_o, status=status)
    torch.cuda.synchronize()
    return table_d.cpu().numpy(), kv.tolist(), rows.cpu().numpy(), int(head_o), status.tolist()


@pytest.mark.parametrize("n_seq,past,new,ps,short", [
    (1, 0, 1, 16, 0), (1, 5, 40, 16, 0), (32, 300, 1, 16, 0), (33, 100, 7, 5, 0), (257, 50, 20, 1, 0), (300, 64, 33, 16, 40),
    (1024, 30, 2, 8, 0), (1025, 200, 50, 24, 100), (6000, 12, 3, 16, 0), (16384, 3, 2, 2, 5000), (3, 0, 9000, 16, 0)])
@pytest.mark.parametrize("alias", [False, True])
def test_plan(gpu, n_seq, past, new, ps, short, alias):
    """Random lengths with idle sequences and full pages, a list that runs out, rows behind the last token."""
    rng = np.random.default_rng(n_seq + past)
    p = rng.integers(0, past + 1, n_seq)
    p[rng.random(n_seq) < 0.2] = past // ps * ps
    n = rng.integers(0, new + 1, n_seq) if new > 1 else np.ones(n_seq, int)
    mp = -(-(past + new) // ps)
    table = np.full((n_seq, mp), -1)
    ids = rng.permutation(n_seq * mp + 4)
    at = 0
    for s in range(n_seq):
        held = -(-p[s] // ps)
        table[s, :held] = ids[at:at + held]
        at += held
    free = ids[at:len(ids)] if not short else ids[at:at + max(1, (n_seq * new // ps) - short) // 2]
    cap = int(n.sum()) + (37 if n_seq % 2 else 0)
    args = (p, n, ps, len(ids), free, 2, table, cap)
    got, want = run_plan(*args, alias=alias), plan_reference(*args)
    for a, b in zip(got, want):
        assert np.array_equal(a, b)


def test_plan_limits(gpu):
    """Negative lengths, sequences past their table, pages outside the cache, too few rows, a free head
    outside the list, sums that stop at 2^31 - 1, no sequence at all."""
    table = np.array([[7, -1, 99], [3, 2**31 - 1, -5], [1, 2, 4], [0, 0, 0]])
    for cap in (0, 3, 200):
        for head in (-4, 0, 2, 50):
            args = ([20, -3, 30, 48], [60, 20, -1, 5], 16, 10, [5, 6, 8, 9], head, table, cap)
            for a, b in zip(run_plan(*args), plan_reference(*args)):
                assert np.array_equal(a, b)
    args = ([2**31 - 1, 2**31 - 5], [7, 100], 16, 4, [1], 0, np.zeros((2, 2), int), 6)
    for a, b in zip(run_plan(*args), plan_reference(*args)):
        assert np.array_equal(a, b)
    rows = torch.full((3, 5), 7, dtype=torch.int32, device="cuda")
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    mc.kv_plan(None, none, 16, 4, none, torch.empty(0, 3, dtype=torch.int32, device="cuda"), rows[0], rows[1], rows[2])
    assert (rows == -1).all()


# ---- the step as it is used ----------------------------------------------------------

def test_decode_steps_in_one_graph(gpu):
    """Planning, norm + rotation + append, attention, routing and the MoE block
    with that routing, captured once and replayed for ten steps of growing
    sequences (one of them idle, a padded row at the end), against a dense
    64-bit attention over everything appended so far."""
    from helpers import small_layer
    E, D, F = 16, 256, 256
    L = small_layer(E, D, F, 2, bias=False, seed_base=11)
    mc.upload_layer(7300, L)
    n_seq, nq, nkv, hd, ps, n_pages, cap, most = 5, 8, 2, 32, 4, 40, 6, 64
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    i32 = dict(dtype=torch.int32, device="cuda")
    past = torch.zeros(n_seq, **i32)
    new = torch.tensor([1, 1, 0, 1, 2], **i32)
    free = torch.randperm(n_pages, generator=g, device="cuda").int()
    head, status = torch.zeros(1, **i32), torch.zeros(3, **i32)
    table = torch.full((n_seq, most // ps), -1, **i32)
    rows = torch.zeros(3, cap, **i32)
    kc, vc = (torch.full((n_pages, ps, nkv, hd), NAN, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    x = torch.zeros(cap, D, device="cuda")
    qkv = torch.zeros(cap, (nq + 2 * nkv) * hd, dtype=torch.bfloat16, device="cuda")
    cut = lambda a, n: qkv[:, a * hd:(a + n) * hd].unflatten(1, (n, hd))  # noqa: E731
    q, k, v = cut(0, nq), cut(nq, nkv), cut(nq + nkv, nkv)
    wq, wk = (1 + 0.2 * torch.randn(hd, generator=g, device="cuda") for _ in range(2))
    rt = rope_table(most, hd)
    qr, o = torch.zeros(cap, nq, hd, dtype=torch.bfloat16, device="cuda"), torch.zeros(cap, nq, hd, dtype=torch.bfloat16, device="cuda")
    ws = torch.empty(mc.paged_attention_workspace(cap, nq, kc, vc, most) + 16, dtype=torch.uint8, device="cuda")
    logits, bias = torch.zeros(cap, E, device="cuda"), 0.1 * torch.randn(E, generator=g, device="cuda")
    idx, p = torch.zeros(cap, 8, **i32), torch.zeros(cap, 8, device="cuda")
    xo = torch.zeros(cap, D, device="cuda")

    def step(s):
        mc.kv_plan(past, new, ps, n_pages, free, table, rows[0], rows[1], rows[2], kv_len=past, free_head=head,
                   free_head_out=head, status=status, stream=s)
        mc.qk_norm_rope(q, k, v, kc, vc, rows[1], rows[2], qr, rope=rt, q_norm=wq, k_norm=wk, stream=s)
        mc.paged_attention(qr, kc, vc, table, rows[1], o, ws, most, hd**-0.5, row_seq=rows[0], stream=s)
        mc.route(logits, idx, p, bias=bias, score="sigmoid", groups=4, keep_groups=3, group_top=2, scale=1.5, stream=s)
        mc.moe_ffn_dev(7300, x, xo, idx, p, flags=mc.GIVEN_TOPK, stream=s)

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step(s)                                          # loads the kernels and grows the layer's workspace
        s.synchronize()
        past.zero_(), head.zero_(), table.fill_(-1), kc.fill_(NAN), vc.fill_(NAN)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            step(torch.cuda.current_stream())
    torch.cuda.synchronize()
    seen = [([], []) for _ in range(n_seq)]
    owner = [0, 1, 3, 4, 4]
    for it in range(10):
        qkv.copy_(torch.randn(qkv.shape, generator=g, device="cuda").bfloat16())
        x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        xo.fill_(1.0)
        logits.copy_(torch.randn(logits.shape, generator=g, device="cuda"))
        o.fill_(4.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        mc.check_status()
        assert rows[0].tolist() == owner + [-1] and int(status[0]) == 5 and int(status[1]) == int(status[2])
        pos = [it, it, it, 2 * it, 2 * it + 1]
        assert rows[1].tolist() == pos + [-1] and past.tolist() == [it + 1, it + 1, 0, it + 1, 2 * it + 2]
        pt = torch.tensor(pos, device="cuda")
        kk, _ = rope_reference(k[:5], wk, 1e-6, rt, pt)
        qq, _ = rope_reference(q[:5], wq, 1e-6, rt, pt)
        assert near(qr[:5], qq, 2.0**-18 * (1 + qq.abs()))
        for r in range(5):
            # the cache holds bf16: what it holds is checked against the 64-bit keys, and the attention goes by it
            sl = int(rows[2, r])
            assert near(kc[sl // ps, sl % ps], kk[r], 2.0**-18 * (1 + kk[r].abs()))
            seen[owner[r]][0].append(kc[sl // ps, sl % ps].clone())
            seen[owner[r]][1].append(v[r].clone())
            assert torch.equal(vc[sl // ps, sl % ps], v[r])
        for r in range(5):
            K = torch.stack(seen[owner[r]][0][:pos[r] + 1]).double().repeat_interleave(nq // nkv, 1)
            V = torch.stack(seen[owner[r]][1][:pos[r] + 1]).double().repeat_interleave(nq // nkv, 1)
            w = torch.softmax(torch.einsum("hd,nhd->hn", qr[r].double(), K) * hd**-0.5, 1)
            want = torch.einsum("hn,nhd->hd", w, V)
            # scores below 2^7: their fp32 errors stay under 2^-12 with the weights' 2^-16
            assert near(o[r], want, 2.0**-12 * torch.einsum("hn,nhd->hd", w, V.abs()))
        assert (o[5] == 4).all()
        sc = torch.sigmoid(logits.double())
        ch = sc + bias.double()
        assert torch.equal(ch.gather(1, idx.long()), ch.gather(1, idx.long()).sort(1, descending=True).values)
        # fp32 weights: the sigmoid errs by 5 units of 2^-24, the sum by as much and 5 additions, quotient and factor by 2
        assert torch.allclose(p.double(), 1.5 * sc.gather(1, idx.long()) / sc.gather(1, idx.long()).sum(1, keepdim=True),
                              rtol=17 * 2.0**-24, atol=0)
        want, _, _ = mc.moe_ffn_host(7300, x.cpu().numpy(), np.ones((cap, D), np.float32),
                                     given=(idx.cpu().numpy(), p.cpu().numpy()))
        assert np.array_equal(xo.cpu().numpy(), want)
    del graph
    mc.free_layer(7300)
