"""GPU: groups whose two summed choices nearly cancel, or overflow in fp32. The
groups that stay have to be those of the 64-bit sums; the reference is
`route_reference`."""
import pytest

from test_gpu_route import check

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups,keep,k", [(64, 32, 16, 8), (64, 16, 5, 6), (256, 8, 4, 8)])
def test_biases_that_cancel_within_a_group(gpu, score, E, groups, keep, k):
    """+1000 and -999.9 as the best two of every group: sums near 0.1, of numbers
    that fp32 rounds to 2^-14. (Where a group has more experts the others are far below.)"""
    g = torch.Generator(device="cuda")
    g.manual_seed(E + groups)
    x = 0.02 * torch.randn(600, E, generator=g, device="cuda")
    if score == "softmax":
        x *= 5
    bias = torch.full((groups, E // groups), -5000.0, device="cuda")
    bias[:, 0], bias[:, 1] = 1000.0, -999.9
    check(x, k, bias.flatten().contiguous(), score, groups, keep, 2)


def test_one_group_of_large_choices_among_ordinary_ones(gpu):
    """The error of a group that is not at the cut counts too: its fp32 sum may
    lie on the wrong side of it."""
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    E, groups = 32, 8
    x = 0.02 * torch.randn(2000, E, generator=g, device="cuda")
    bias = 0.01 * torch.randn(groups, E // groups, generator=g, device="cuda")
    bias[3] = -9000.0
    bias[3, 0], bias[3, 2] = 4000.0, -3999.0            # 1 and both scores: among the others' sums
    check(x, 6, bias.flatten().contiguous(), "sigmoid", groups, 4, 2)


def test_sums_that_overflow_fp32(gpu):
    """Biases near fp32's largest: sums of two are infinite there, not in 64 bits."""
    E, groups = 16, 4
    x = torch.zeros(1, E)
    bias = torch.zeros(groups, E // groups)
    bias[0, 0], bias[0, 1] = 2.0e38, 2.0e38
    bias[2, 0], bias[2, 1] = 3.0e38, 3.0e38
    bias[3, 1], bias[3, 3] = 2.5e38, 2.5e38
    idx, _ = check(x.cuda(), 4, bias.flatten().contiguous().cuda(), "sigmoid", groups, 2, 2)
    assert sorted(idx[0].tolist()) == [8, 9, 13, 15]
