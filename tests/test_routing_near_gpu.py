"""Routing from logits where float32 keys leave the order open, in rows of every
width and batches that fill a warp's rows or do not, on the GPU, against the plain
implementation in 64 bits of test_routing_gpu.py (ids equal)."""
import numpy as np
import pytest

from test_routing_gpu import check_route, plain_scores

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("E", [3, 8, 13, 16, 32, 60, 64, 128, 256])
def test_rows_that_leave_the_order_open(cuda, E, masked, score):
    """Logits on a coarse grid with biases that undo one row's scores to float32: keys
    next to zero whose order is that of the biases' roundings, beside rows that are
    decided and rows with few experts."""
    import torch
    from aethermoe_b200 import routing
    g = torch.Generator(device=cuda)
    g.manual_seed(E)
    for T in (1, 2, 3, 7, 33, 40, 300):
        x = (2 * torch.randn(T, E, device=cuda, generator=g)).round() / 2
        if masked:
            x[torch.rand(T, E, device=cuda, generator=g) < 0.5] = -np.inf
        at = T // 2
        s = plain_scores(x[at:at + 1].double().cpu().numpy(), score)[0]
        bias = torch.from_numpy(-s.astype(np.float32)).to(cuda)
        for dt in (torch.float32, torch.bfloat16):
            for k in {1, min(2, E), min(5, E), min(7, E), min(8, E)}:
                for groups, top, gt in ((1, 1, 1), (4, 2, 2)):
                    if E % groups or k > E // groups * top:
                        continue
                    how = dict(k=k, score=score, groups=groups, top_groups=top, group_top=gt)
                    ids, w = routing.route_tokens(x.to(dt), bias=bias, **how)
                    check_route(x.to(dt), ids, w, dict(how, bias=bias.cpu().numpy()))
