"""Routing from logits where masks leave fewer experts than slots, and NaN among
the biases, on the GPU, against the plain implementation in 64 bits of
test_routing_gpu.py (ids equal, weights within its bound)."""
import numpy as np
import pytest

from test_routing_gpu import check_route, make

pytestmark = pytest.mark.gpu

# groups of whole lanes of 8 experts, one and more of them, for every width of a
# row, then groups of other sizes
GROUPS = [(16, 2, 1), (24, 3, 1), (32, 4, 2), (64, 8, 4), (64, 4, 3), (128, 16, 5), (128, 8, 3), (256, 8, 4),
          (256, 16, 8), (256, 32, 2), (60, 4, 2), (96, 4, 2), (8, 4, 2), (250, 10, 3)]


@pytest.mark.parametrize("E,groups,top", GROUPS)
def test_groups_with_fewer_experts_than_slots(cuda, E, groups, top):
    """Rows whose kept groups have no, one or two experts left: the other slots are
    empty, whatever the dropped groups, before and behind the kept ones, still have."""
    import torch
    from aethermoe_b200 import routing
    size, T = E // groups, 33
    rng = np.random.default_rng(E + groups)
    x = rng.uniform(-3.0, -2.0, (T, E))
    for t in range(T):
        for g in rng.choice(groups, top, replace=False):
            x[t, g * size:(g + 1) * size] = -np.inf
            on = rng.choice(size, min(size, t % 3), replace=False)
            x[t, g * size + on] = rng.uniform(4.0, 6.0, len(on))
    x[T - 1] = -np.inf
    x = torch.from_numpy(x).to(cuda)
    bias = 0.01 * torch.randn(E, device=cuda)
    for dt in (torch.float32, torch.bfloat16):
        for k in (4, 8):
            if k > size * top:
                continue
            for score in ("softmax", "sigmoid"):
                for b in (None, bias):
                    for group_top in (1, 2):
                        for renorm in (False, True):
                            how = dict(k=k, score=score, groups=groups, top_groups=top, group_top=group_top,
                                       renormalize=renorm)
                            ids, w = routing.route_tokens(x.to(dt), bias=b, **how)
                            check_route(x.to(dt), ids, w, dict(how, bias=None if b is None else b.cpu().numpy()))


@pytest.mark.parametrize("E,groups,top", GROUPS)
def test_biases_that_leave_fewer_experts_than_slots(cuda, E, groups, top):
    """The same where the biases, alike for all rows, take the experts out."""
    import torch
    from aethermoe_b200 import routing
    size = E // groups
    x = make(cuda, 40, E, torch.float32, seed=E)
    for left in (0, 1, 2):
        bias = torch.full((E,), -np.inf, device=cuda)
        for g in range(groups):
            if g % 2:  # full, but with small keys
                bias[g * size:(g + 1) * size] = -4.0
            else:
                bias[g * size:g * size + min(left, size)] = 1.0
        for score in ("softmax", "sigmoid"):
            for group_top in (1, 2):
                how = dict(k=min(4, size * top), score=score, groups=groups, top_groups=top, group_top=group_top)
                ids, w = routing.route_tokens(x, bias=bias, **how)
                check_route(x, ids, w, dict(how, bias=bias.cpu().numpy()))

@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [False, True])
def test_nan_bias(cuda, score, renorm):
    """A NaN among the biases ranks its expert first; the weight is that of its score."""
    import torch
    from aethermoe_b200 import routing
    for E in (8, 24, 64, 256):
        x = make(cuda, 20, E, torch.float32, seed=E)
        bias = 0.1 * torch.randn(E, device=cuda)
        bias[5] = np.nan
        for groups, top, gt in ((1, 1, 1), (4, 2, 2), (4, 2, 1)):
            how = dict(k=3, score=score, groups=groups, top_groups=top, group_top=gt, renormalize=renorm)
            ids, w = routing.route_tokens(x, bias=bias, **how)
            assert (ids[:, 0] == 5).all() and torch.isfinite(w).all()
            check_route(x, ids, w, dict(how, bias=bias.cpu().numpy()))
