"""CPU: what the paged-cache attention and routing entry points refuse. Every
argument is checked before any CUDA call, so the refusals show without a GPU;
the pointers here are never read."""
import ctypes as C

import numpy as np
import pytest

import moe_cuda as mc

DEALT = 512                   # rows whose work is dealt evenly
P = 0x7000_0000_0000          # a 16-byte aligned address that nothing reads
INVALID, UNSUPPORTED = mc.MOE_ERR_INVALID, mc.MOE_ERR_UNSUPPORTED


def cache(**over):
    d = dict(k=P, v=P, dtype=mc.BF16, n_pages=8, page_size=16, n_kv=2, head_dim=64, page_stride=16 * 128,
             token_stride=128, head_stride=64)
    d.update(over)
    return mc.MoeKvCache(**d)


def plan(**over):
    d = dict(past=P, new=P, n_seq=4, page_size=16, n_pages=64, free=P, n_free=8, head=P, table=P, max_pages=8, kv=P,
             seq=P, pos=P, slot=P, cap=8, head_out=P, status=P)
    d.update(over)
    return mc.lib().moe_kv_plan_dev(*d.values(), None)


def rope(c=None, **over):
    d = dict(q=P, ldq=256, k=P, ldk=128, v=P, ldv=128, dtype=mc.BF16, rows=4, n_q=4, qn=P, kn=P, eps=1e-6, rope=P, rot=64,
             n_rope=100, pos=P, slot=P, out=P + (1 << 20), ldo=256)
    d.update(over)
    return mc.lib().moe_qk_norm_rope_dev(*d.values(), C.byref(c or cache()), None)


def attn(c=None, **over):
    c = c or cache()
    d = dict(q=P, ldq=256, cache=C.byref(c), table=P, n_seq=4, max_pages=8, seq=None, pos=P, rows=4, n_q=4, max_kv=4096,
             scale=0.1, out=P, ldo=256, lse=None, ws=P, n=1 << 30)
    d.update(over)
    return mc.lib().moe_paged_attention_dev(*d.values(), None)


def route(**over):
    d = dict(x=P, ld=64, dtype=mc.F32, rows=4, E=64, bias=None, score=0, groups=4, keep=2, top=2, k=8, renorm=1, factor=1.0,
             idx=P, p=P)
    d.update(over)
    return mc.lib().moe_route_dev(*d.values(), None)


@pytest.mark.parametrize("over,want", [
    (dict(n_seq=-1), INVALID), (dict(cap=-1), INVALID), (dict(n_free=-1), INVALID), (dict(page_size=0), INVALID),
    (dict(max_pages=0), INVALID), (dict(n_pages=0), INVALID), (dict(new=None), INVALID), (dict(table=None), INVALID),
    (dict(free=None), INVALID), (dict(seq=None), INVALID), (dict(slot=None), INVALID), (dict(n_seq=16385), UNSUPPORTED),
    (dict(n_pages=1 << 20, page_size=1 << 11), UNSUPPORTED), (dict(max_pages=1 << 30), UNSUPPORTED)])
def test_plan_refuses(over, want):
    assert plan(**over) == want and b"moe_kv_plan_dev" in mc.lib().moe_cuda_last_error()


def test_empty_calls_do_nothing():
    assert plan(n_seq=0, cap=0, head_out=None, status=None) == mc.MOE_OK
    assert rope(rows=0) == mc.MOE_OK and rope(n_q=0, q=None, out=None, slot=None) == mc.MOE_OK
    assert attn(rows=0) == mc.MOE_OK
    assert route(rows=0) == mc.MOE_OK


BAD_CACHES = [(dict(k=None), INVALID), (dict(dtype=mc.Q8), INVALID), (dict(n_pages=0), INVALID), (dict(page_size=0), INVALID),
              (dict(n_kv=0), INVALID), (dict(head_dim=12), UNSUPPORTED), (dict(head_dim=264), UNSUPPORTED),
              (dict(head_dim=0), UNSUPPORTED), (dict(k=P + 8), INVALID), (dict(token_stride=132), INVALID),
              (dict(page_stride=-2048), INVALID), (dict(n_pages=1 << 20, page_size=1 << 11), UNSUPPORTED)]


@pytest.mark.parametrize("over,want", BAD_CACHES)
def test_bad_caches_are_refused(over, want):
    assert rope(cache(**over)) == want
    assert attn(cache(**over)) == want
    assert mc.lib().moe_paged_attention_workspace(4, 4, C.byref(cache(**over)), 128) == 0


@pytest.mark.parametrize("over,want", [
    (dict(dtype=7), INVALID), (dict(dtype=mc.F16), UNSUPPORTED), (dict(rows=-1), INVALID), (dict(q=None), INVALID),
    (dict(out=None), INVALID), (dict(k=None), INVALID), (dict(rot=72), UNSUPPORTED), (dict(rot=12), UNSUPPORTED),
    (dict(rope=None), INVALID), (dict(n_rope=0), INVALID), (dict(pos=None), INVALID), (dict(eps=-1.0), INVALID),
    (dict(eps=float("nan")), INVALID), (dict(ldq=255), INVALID), (dict(ldo=128), INVALID), (dict(ldq=260), INVALID),
    (dict(q=P + 8), INVALID), (dict(ldk=132), INVALID), (dict(qn=P + 4), INVALID), (dict(rope=P + 8), INVALID),
    (dict(out=P + 512), INVALID),                                          # overlaps q, is not q
    (dict(out=P, ldo=512), INVALID),                                       # q, but another stride
    (dict(q=P + (1 << 21), out=P), INVALID)])                              # overlaps k
def test_rope_refuses(over, want):
    assert rope(**over) == want


@pytest.mark.parametrize("over", [
    dict(out=P + 512), dict(out=P, ldo=512), dict(out=P + 1024, ldq=512, ldo=512 + 64), dict(ldq=480, out=P + 512, ldo=480)])
def test_attention_refuses_an_output_across_its_queries(over):
    """Rows of 512 bytes: another offset, another stride, columns that meet at
    either end."""
    assert attn(**over) == INVALID and b"overlaps q" in mc.lib().moe_cuda_last_error()


@pytest.mark.parametrize("over,want", [
    (dict(rows=-1), INVALID), (dict(n_q=3), INVALID), (dict(n_q=0), INVALID), (dict(n_q=32770), UNSUPPORTED), (dict(n_seq=-1), INVALID),
    (dict(max_pages=0), INVALID), (dict(rows=5), INVALID), (dict(max_kv=0), INVALID), (dict(q=None), INVALID),
    (dict(out=None), INVALID), (dict(pos=None), INVALID), (dict(table=None), INVALID), (dict(ldq=128), INVALID),
    (dict(ldo=260), INVALID), (dict(q=P + 2), INVALID), (dict(ws=None), INVALID), (dict(ws=P + 8), INVALID),
    (dict(n=64), INVALID)])
def test_attention_refuses(over, want):
    assert attn(**over) == want and b"moe_paged_attention_dev" in mc.lib().moe_cuda_last_error()


def test_attention_workspace_size():
    """None for contexts up to 2048 positions (one launch); above, a row of
    head_dim + 2 floats per query head and 64 positions (512 where rows are too
    many to be dealt out), at most 128."""
    ws = mc.lib().moe_paged_attention_workspace
    for rows, n_q, max_kv in ((1, 2, 1), (4, 4, 64), (1, 32, 2048), (600, 4, 1000), (0, 4, 4096), (4, 3, 4096), (4, 4, 0)):
        assert ws(rows, n_q, C.byref(cache()), max_kv) == 0
    for rows, n_q, max_kv in ((1, 2, 2049), (1, 32, 1 << 20), (33, 8, 8192), (600, 4, 5000), (1, 2, 2**31 - 1)):
        n = ws(rows, n_q, C.byref(cache()), max_kv)
        one = rows * n_q * (64 + 2) * 4
        assert n == min(128, -(-max_kv // (64 if rows <= DEALT else 512))) * one + 16


@pytest.mark.parametrize("over,want", [
    (dict(dtype=mc.Q4), INVALID), (dict(rows=-1), INVALID), (dict(E=0), INVALID), (dict(ld=63), INVALID),
    (dict(E=1028, ld=1028), UNSUPPORTED), (dict(score=2), INVALID), (dict(groups=0), INVALID), (dict(groups=5), INVALID),
    (dict(keep=5), INVALID), (dict(keep=0), INVALID), (dict(groups=64, keep=64), UNSUPPORTED), (dict(top=3), INVALID),
    (dict(k=0), INVALID), (dict(k=33, groups=1, keep=1), UNSUPPORTED), (dict(k=17, groups=8, keep=2), INVALID),
    (dict(x=None), INVALID), (dict(idx=None), INVALID), (dict(p=None), INVALID)])
def test_route_refuses(over, want):
    assert route(**over) == want and b"moe_route_dev" in mc.lib().moe_cuda_last_error()


def test_binding_refuses_host_tensors_and_wrong_types():
    torch = pytest.importorskip("torch")
    k = torch.zeros(2, 16, 2, 64)
    i = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: mc.paged_attention(torch.zeros(2, 4, 64), k, k, torch.zeros(2, 1, dtype=torch.int32), i,
                                            torch.zeros(2, 4, 64), None, 16, 1.0),
                 lambda: mc.qk_norm_rope(None, k[0], k[0], k, k, None, i, None),
                 lambda: mc.kv_plan(i, i, 16, 2, i, torch.zeros(2, 1, dtype=torch.int32), i, i, i),
                 lambda: mc.route(torch.zeros(2, 8), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, 2)),
                 lambda: mc.kv_cache(k, k.transpose(1, 2)), lambda: mc.kv_cache(k.int(), k.int())):
        with pytest.raises(mc.MoeError):
            call()


def test_binding_arguments():
    """Positions and keywords as documented; unknown, double and missing ones are a TypeError, as of a Python function."""
    torch = pytest.importorskip("torch")
    for f in (mc.kv_plan, mc.qk_norm_rope, mc.paged_attention, mc.route):
        assert f.__doc__ and f.__name__ in f.__doc__
        with pytest.raises(TypeError):
            f()
        with pytest.raises(TypeError):
            f(*range(20))
    x, i, p = torch.zeros(2, 8), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, 2)
    with pytest.raises(TypeError):
        mc.route(x, i, p, experts=3)
    with pytest.raises(TypeError):
        mc.route(x, i, p, topk_p=p)
    for bad in ((None, i, p), (3, i, p), (x, "i", p), (x.double(), i, p), (x, i.long(), p)):
        with pytest.raises(mc.MoeError) as e:
            mc.route(*bad)
        assert e.value.code == INVALID
    assert not hasattr(mc, "no_such_call")


def test_page_division_by_multiplication():
    """The kernels divide positions by the page size with one multiply; the
    same arithmetic here, at the quotients' edges, for every page size that
    could go wrong first (small ones, powers of two and their neighbours)."""
    rng = np.random.default_rng(0)
    for d in sorted({*range(1, 300), *(max(1, (1 << b) + o) for b in range(31) for o in (-1, 0, 1))}):
        if d > 2**31 - 1:
            continue
        l = (d - 1).bit_length()
        m = (1 << (31 + l)) // d + 1
        assert m < 1 << 32
        top = (2**31 - 1) // d
        for q in {0, 1, top, top - 1, *rng.integers(0, top + 1, 20).tolist()}:
            for n in (q * d - 1, q * d, q * d + d - 1):
                if 0 <= n < 2**31:
                    assert (n * m) >> (31 + l) == n // d


def test_pieces_are_dealt_whole_and_in_few_parts():
    """The arithmetic by which the attention deals the rows' 64-position pieces
    to groups of CTAs: every piece to one group, a row's groups in succession
    and no more of them than it has room for, shares equal to a piece."""
    rng = np.random.default_rng(1)
    for _ in range(400):
        rows = int(rng.integers(1, 40))
        pieces = rng.integers(0, int(2 ** rng.uniform(0, 12)) + 1, rows)
        parts, grid = int(rng.integers(33, 129)), int(rng.integers(1, 150))
        total, most = int(pieces.sum()), int(pieces.max())
        if total == 0:
            continue
        G = min(grid, total)
        if most > 1:
            G = min(G, max(1, (parts - 1) * total // (most - 1)))
        cuts = [g * total // G for g in range(G + 1)]
        assert cuts[0] == 0 and cuts[-1] == total and {b - a for a, b in zip(cuts, cuts[1:])} <= {total // G, -(-total // G)}
        owner = np.searchsorted(np.array(cuts), np.arange(total), side="right") - 1
        assert all(((x + 1) * G - 1) // total == owner[x] for x in range(total))
        base = 0
        for u in pieces.tolist():
            if u:
                first, last = ((base + 1) * G - 1) // total, ((base + u) * G - 1) // total
                assert last - first + 1 <= parts
            base += u


def test_host_driver_without_a_gpu_keeps_its_cpu_caches():
    """mh_kv_device refuses bad arguments, and where there is no GPU fails
    loudly; the model's CPU attention then works as before."""
    mh = pytest.importorskip("moe_host")
    torch = pytest.importorskip("torch")
    from helpers import TINY, tiny_model
    g, attn, _ = tiny_model(2, seed=1)
    m = mh.HostModel(TINY, batch=1, max_ctx=8)
    m.set_globals(g["tok_emb"], g["final_norm_w"], g["lm_head"])
    for l, a in enumerate(attn):
        m.set_layer(l, a)
    for args in ((9, 16), (mc.F32, 0)):
        with pytest.raises(mc.MoeError) as e:
            m.kv_device(*args)
        assert e.value.code == INVALID
    if not torch.cuda.is_available():
        with pytest.raises(mc.MoeError):
            m.kv_device(mc.F32, 16)
    x = np.ones((2, TINY["d_model"]), np.float32)
    assert np.isfinite(m.attention(0, x, 2)[0]).all()
    m.close()
