"""GPU: routing by groups where scores say less than logits do. Without a bias
the experts of the kept groups are ordered by their logits, which order the
exact scores however close those lie; groups are chosen by sums of scores in
64 bits, also where the two that are summed cancel."""
import math

import numpy as np
import pytest

import moe_cuda as mc

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def by_logit_reference(x, score, groups, keep, group_top, k):
    """Experts by logit within the groups that 64-bit scores keep."""
    T, E = x.shape
    size = E // groups
    x = x.astype(np.float64)
    out = np.full((T, k), -1, np.int32)
    for t in range(T):
        s = np.exp(x[t] - x[t].max())
        s = s / s.sum() if score == "softmax" else 1 / (1 + np.exp(-x[t]))
        best = [sum(sorted(s[g * size:(g + 1) * size])[::-1][:group_top]) for g in range(groups)]
        stay = sorted(range(groups), key=lambda g: -best[g])[:keep]
        mine = [e for e in range(E) if e // size in stay]
        out[t] = sorted(mine, key=lambda e: -x[t, e])[:k]
    return out


def chosen(x, k, **kw):
    idx = torch.full((x.shape[0], k), 77, dtype=torch.int32, device="cuda")
    p = torch.full((x.shape[0], k), 77.0, device="cuda")
    mc.route(x, idx, p, **kw)
    torch.cuda.synchronize()
    return idx.cpu().numpy(), p.cpu().numpy()


@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("group_top", [1, 2])
def test_saturated_sigmoids_are_ordered_by_logit(gpu, dt, group_top):
    """Logits of 40 and more all have the 64-bit score 1."""
    x = torch.full((1, 32), -4.0)
    x[0, 3], x[0, 5], x[0, 6], x[0, 17] = 40.0, 50.0, 45.0, 60.0
    idx, p = chosen(x.to(dt).cuda(), 4, score="sigmoid", groups=4, keep_groups=2, group_top=group_top, renorm=False)
    assert idx[0].tolist() == [17, 5, 6, 3]
    assert (p == 1).all()


def test_neighbouring_logits_with_one_score(gpu):
    """25 and the next fp32 number have sigmoids that differ by 2^-56: one 64-bit number."""
    x = torch.full((1, 16), -1.0)
    x[0, 1] = 25.0
    x[0, 2] = float(np.nextafter(np.float32(25), np.float32(30)))
    idx, _ = chosen(x.cuda(), 2, score="sigmoid", groups=2, keep_groups=1, group_top=1)
    assert idx[0].tolist() == [2, 1]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=str)
def test_softmax_scores_that_underflow(gpu, dt):
    """Logits 800 and more below the largest: softmax scores of 0 in 64 bits."""
    x = torch.full((1, 16), -960.0)
    x[0, 1], x[0, 4], x[0, 5], x[0, 6] = 0.0, -900.0, -800.0, -840.0
    idx, p = chosen(x.to(dt).cuda(), 4, score="softmax", groups=2, keep_groups=1, group_top=2)
    assert idx[0].tolist() == [1, 5, 6, 4] and p[0].tolist() == [1, 0, 0, 0]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups,keep,group_top,k", [(256, 8, 4, 2, 8), (64, 8, 3, 1, 6), (1024, 32, 2, 2, 32)])
def test_many_tokens_of_large_logits(gpu, score, E, groups, keep, group_top, k):
    """Thousands of tokens whose scores crowd at one (sigmoid) or at zero
    (softmax); the groups' sums stay apart, each group having its own level."""
    g = torch.Generator(device="cuda")
    g.manual_seed(E)
    T = 1000
    level = torch.stack([torch.randperm(groups, generator=g, device="cuda") for _ in range(T)]).float()
    x = 30 + 3 * torch.randn(T, E, generator=g, device="cuda").abs() if score == "sigmoid" else \
        -700 - 100 * torch.rand(T, E, generator=g, device="cuda")
    x = x.view(T, groups, -1)
    # two experts of each group decide about it
    x[:, :, 1], x[:, :, 2] = (level * 0.2 - 3, level * 0.1 - 3) if score == "softmax" else (x[:, :, 1], x[:, :, 2])
    if score == "sigmoid":                      # a group of low logits where it is to be left out
        x = torch.where((level < keep)[:, :, None], x, x - 33)
    x = x.reshape(T, E).contiguous()
    idx, _ = chosen(x, k, score=score, groups=groups, keep_groups=keep, group_top=group_top)
    assert np.array_equal(idx, by_logit_reference(x.cpu().numpy(), score, groups, keep, group_top, k))
