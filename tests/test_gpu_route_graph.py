"""GPU: routing captured into a graph and replayed over new logits: the chosen
experts are the best each time (not only in order), and what it leaves empty
adds nothing in the MoE block that takes its lists."""
import math

import numpy as np
import pytest

import moe_cuda as mc
from helpers import small_layer
from test_gpu_route import route_reference

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("score,biased,groups,keep", [("sigmoid", True, 4, 3), ("sigmoid", False, 4, 2), ("softmax", False, 1, 1)])
@pytest.mark.parametrize("T", [1, 6, 40])
def test_replayed_routing_into_the_moe_block(gpu, score, biased, groups, keep, T):
    E, D, k, lid = 16, 256, 8, 7310
    mc.upload_layer(lid, small_layer(E, D, 256, 2, bias=False, seed_base=12))
    g = torch.Generator(device="cuda")
    g.manual_seed(T)
    x, xo, logits = torch.zeros(T, D, device="cuda"), torch.zeros(T, D, device="cuda"), torch.zeros(T, E, device="cuda")
    bias = 0.1 * torch.randn(E, generator=g, device="cuda") if biased else None
    idx, p = torch.zeros(T, k, dtype=torch.int32, device="cuda"), torch.zeros(T, k, device="cuda")

    def step(s):
        mc.route(logits, idx, p, bias=bias, score=score, groups=groups, keep_groups=keep, group_top=2, scale=1.5, stream=s)
        mc.moe_ffn_dev(lid, x, xo, idx, p, flags=mc.GIVEN_TOPK, stream=s)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(s)                                          # loads the kernels and grows the layer's workspace
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            step(torch.cuda.current_stream())
    torch.cuda.synchronize()
    for it in range(8):
        x.copy_(torch.randn(T, D, generator=g, device="cuda"))
        xo.fill_(1.0)
        new = torch.randn(T, E, generator=g, device="cuda")
        if it % 2:                                       # too few experts left: empty places in the lists
            new[T // 2, 2 + it:] = math.nan
            new[T - 1, :] = -math.inf
        logits.copy_(new)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        mc.check_status()
        want, wp = route_reference(new.cpu().numpy(), None if bias is None else bias.cpu().numpy(), score, groups, keep, 2, k, True, 1.5)
        got = idx.cpu().numpy()
        assert np.array_equal(got, want)
        assert (np.abs(p.cpu().numpy() - wp) <= 32 * 2.0**-24 * wp).all()     # |logits| < 6: 2 (6 + 5) + 5 + 2 units of 2^-24
        out, _, _ = mc.moe_ffn_host(lid, x.cpu().numpy(), np.ones((T, D), np.float32), given=(got, p.cpu().numpy()))
        assert np.array_equal(xo.cpu().numpy(), out)
        for t in range(T):
            if (got[t] < 0).all():
                assert (xo[t] == 1).all()
    del graph
    mc.free_layer(lid)
