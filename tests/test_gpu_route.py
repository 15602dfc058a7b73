"""GPU: expert routing from given logits against a plain 64-bit form. The
chosen experts have to be equal. A weight is computed in fp32, in units of
2^-24: exp errs by 4 (2 ulp) and by z, its rounded argument (x minus the
largest chosen, or of all, logit), a sigmoid by 5; the sum it is divided by by
as much, and by its additions (5 over the warp, 32 more and the mean of z, below
8, where it runs over all experts); the quotient and the factor by 2."""
import math

import numpy as np
import pytest

import moe_cuda as mc

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def route_reference(x, bias, score, groups, keep, group_top, k, renorm, factor):
    T, E = x.shape
    x = x.astype(np.float64)
    idx, p = np.full((T, k), -1, np.int32), np.zeros((T, k))
    size = E // groups
    for t in range(T):
        here = ~np.isnan(x[t]) & (x[t] > -np.inf)
        s = np.zeros(E)
        if here.any():
            if score == "softmax":
                top = x[t][here].max()
                with np.errstate(invalid="ignore"):
                    e = np.where(here, np.where(x[t] == top, 1.0, np.exp(x[t] - top)), 0.0)
                s = e / e.sum()
            else:
                with np.errstate(over="ignore"):
                    s = np.where(here, 1 / (1 + np.exp(-x[t])), 0.0)
        c = s.copy() if bias is None else s + bias.astype(np.float64)
        here &= ~np.isnan(c) & (c > -np.inf)
        allowed = here.copy()
        if keep < groups:
            best = [(sum(sorted(c[g * size:(g + 1) * size][here[g * size:(g + 1) * size]])[::-1][:group_top])
                     if here[g * size:(g + 1) * size].any() else -math.inf) for g in range(groups)]
            stay = sorted(range(groups), key=lambda g: -best[g])[:keep]
            for g in range(groups):
                if g not in stay:
                    allowed[g * size:(g + 1) * size] = False
        rank = x[t] if bias is None and keep == groups else c
        order = sorted(np.flatnonzero(allowed), key=lambda e: -rank[e])[:k]
        idx[t, :len(order)] = order
        w = s[order]
        if renorm:
            w = w / w.sum() if w.sum() > 0 else w * 0
        p[t, :len(order)] = w * factor
    return idx, p


def check(x, k, bias=None, score="softmax", groups=1, keep=1, group_top=1, renorm=True, factor=1.0):
    T, E = x.shape
    idx = torch.full((T, k), 77, dtype=torch.int32, device="cuda")
    p = torch.full((T, k), 77.0, device="cuda")
    mc.route(x, idx, p, bias=bias, score=score, groups=groups, keep_groups=keep, group_top=group_top, renorm=renorm, scale=factor)
    torch.cuda.synchronize()
    want_i, want_p = route_reference(x.float().cpu().numpy(), None if bias is None else bias.cpu().numpy(), score, groups, keep,
                                     group_top, k, renorm, factor)
    assert np.array_equal(idx.cpu().numpy(), want_i)
    xs = np.take_along_axis(x.double().cpu().numpy(), np.maximum(want_i, 0).astype(np.int64), 1)
    seen = np.where((want_i >= 0) & np.isfinite(xs), xs, -np.inf)
    high = np.where(np.isnan(x.double().cpu().numpy()), -np.inf, x.double().cpu().numpy()).max(1, keepdims=True) \
        if score == "softmax" and not renorm else seen.max(1, keepdims=True)
    with np.errstate(invalid="ignore"):
        z = np.nan_to_num(np.clip(high - seen, 0, 1e4), nan=0.0, posinf=1e4).max(1, keepdims=True)
    units = 2 * (z + 5) + (45 if not renorm else 5) + 2
    err = np.abs(p.cpu().numpy() - want_p) - units * 2.0**-24 * np.abs(want_p) - factor * 2.0**-126
    assert (err <= 0).all(), float(err.max())
    return idx, p


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,k,groups,keep,group_top,biased,renorm", [
    (1, 128, 8, 1, 1, 1, False, True), (16, 128, 8, 1, 1, 1, False, False), (33, 256, 8, 8, 4, 2, True, True),
    (7, 60, 4, 1, 1, 1, True, False), (5, 1, 1, 1, 1, 1, False, True), (3, 2, 2, 1, 1, 1, True, True),
    (9, 8, 8, 4, 4, 2, True, True), (301, 160, 6, 20, 3, 1, False, True), (10, 512, 10, 32, 2, 2, True, False),
    (4, 1024, 32, 1, 1, 1, True, True), (6, 1000, 32, 8, 1, 1, False, False), (11, 33, 5, 3, 2, 2, False, True),
    (2000, 64, 6, 8, 3, 1, True, True), (5, 24, 3, 24, 5, 2, False, False)])
def test_route(gpu, dt, score, T, E, k, groups, keep, group_top, biased, renorm):
    g = torch.Generator(device="cuda")
    g.manual_seed(T * E)
    x = (2 * torch.randn(T, E, generator=g, device="cuda")).to(dt)
    bias = 0.2 * torch.randn(E, generator=g, device="cuda") if biased else None
    check(x, k, bias, score, groups, keep, group_top, renorm, 2.5)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,keep,biased", [(1, 1, False), (1, 1, True), (4, 2, True), (4, 2, False)])
def test_ties_and_masked_experts(gpu, score, groups, keep, biased):
    """Equal logits go to the lower index; NaN and -inf are never chosen, and
    too few experts leave -1 and 0; +inf, the type's lowest value, signed zeros."""
    E, k = 16, 6
    low = torch.finfo(torch.float32).min
    nan, inf = math.nan, math.inf
    x = torch.zeros(9, E)
    x[1, 3::4] = 1.0
    x[2] = nan
    x[3] = -inf
    x[4, :] = -inf
    x[4, 9], x[4, 2] = 0.5, 0.25
    x[5, ::2] = nan
    x[6] = low
    x[6, 11] = -5.0
    x[7, 1::2] = -0.0
    x[8] = torch.arange(E) * 3.0 - 20
    x[8, 5] = nan
    bias = None
    if biased:
        bias = torch.zeros(E)
        bias[4], bias[7], bias[10] = nan, -inf, 0.25
        bias = bias.cuda()
    check(x.cuda(), k, bias, score, groups, keep, 2, True)
    check(x.cuda(), k, bias, score, groups, keep, 1, False)
    if score == "sigmoid" or groups == 1:
        x = x[:1].clone()
        x[0, 6] = inf
        check(x.cuda(), k, bias, score, groups, keep, 1, True)


def test_near_ties_are_ordered_in_64_bits(gpu):
    """Sigmoid scores that round to the same fp32 number still differ."""
    x = torch.full((1, 64), 9.0)
    x[0, 50], x[0, 20], x[0, 63] = 9.00001, 9.00002, 8.99999
    for bias in (None, torch.full((64,), 3.0).cuda()):
        idx, _ = check(x.cuda(), 3, bias, "sigmoid")
        assert idx[0].tolist() == [20, 50, 0]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_many_tokens_choose_as_64_bits_do(gpu, score):
    """A balance bias over scores that lie close: thousands of tokens, some of
    which fp32 cannot rank."""
    g = torch.Generator(device="cuda")
    g.manual_seed(6)
    x = 0.02 * torch.randn(3000, 256, generator=g, device="cuda")
    check(x, 8, 0.001 * torch.randn(256, generator=g, device="cuda"), score, 8, 4, 2)
    check(x[:500], 8, None, score, 8, 4, 2)
    check(x[:500] + 12, 8, torch.zeros(256, device="cuda"), score, 1, 1, 1)


def test_ratios_survive_where_scores_underflow(gpu):
    x = torch.full((2, 32), -300.0)
    x[0, 3], x[0, 4], x[1, 5] = -299.0, -299.5, 200.0
    y = torch.full((2, 32), -91.0)
    y[0, 3], y[1, 5], y[1, 6] = -10.0, 1.0, -70.0      # some of the chosen underflow, their share does not
    for score in ("sigmoid", "softmax"):
        check(x.cuda(), 4, None, score)
        check(y.cuda(), 6, None, score)
    bias = torch.zeros(32)
    bias[8:12] = 5.0                                # the chosen are not the likely ones
    check(x.cuda(), 4, bias.cuda(), "softmax")


def test_strided_rows_another_stream_and_repeat(gpu):
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    wide = torch.randn(50, 200, generator=g, device="cuda")
    idx, p = check(wide[:, 3:131], 8)
    s = torch.cuda.Stream()
    i2, p2 = torch.empty_like(idx), torch.empty_like(p)
    s.wait_stream(torch.cuda.current_stream())
    mc.route(wide[:, 3:131], i2, p2, stream=s)
    s.synchronize()
    assert torch.equal(idx, i2) and torch.equal(p, p2)
