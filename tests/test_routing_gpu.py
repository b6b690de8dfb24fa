"""Routing from logits and its gradient on the GPU, against a plain implementation
in 64 bits.

Ids are equal: the choice is defined by 64-bit keys.  A weight is off by, in
units of 2^-24 of itself: exp (2 ulp: 4) and its argument's rounding (|x - m|),
the sum's terms (5 and 13 additions), the reciprocal and the product (2), the
renormalising sum (k) and quotient with scale (4), twice for numerator and
denominator: under 40 + 2 k + |x - m|.  A gradient is at most twice that off,
relative to the magnitudes of the terms that it is a difference of, and has k more
additions: 2 (40 + 2 k + |x - m|) + k.  bf16 gradients add 2^-8 of their value.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U32, HALF_BF16 = 2.0 ** -24, 2.0 ** -8


def plain_scores(x, score):
    with np.errstate(all="ignore"):
        if score == "sigmoid":
            t = np.exp(-np.abs(x))
            return np.where(x < 0, t, 1.0) / (1 + t)
        m = np.where(np.isnan(x), -np.inf, x).max(1, keepdims=True)
        e = np.exp(x - np.where(m == -np.inf, 0.0, m))
        z = e.sum(1, keepdims=True)
        return np.where(z == 0, 0.0, e / z)


def in_order(keys, n):
    """Indices of the n largest, NaN first, ties to the lower index, -inf never."""
    at = [i for i in range(len(keys)) if not keys[i] == -np.inf]
    at.sort(key=lambda i: (not np.isnan(keys[i]), 0.0 if np.isnan(keys[i]) else -keys[i], i))
    return at[:n]


def plain_route(x, k, score="softmax", bias=None, groups=1, top_groups=1, group_top=1, renormalize=False, scale=1.0):
    """(ids, weights, scores) in 64 bits."""
    x = np.asarray(x, np.float64)
    T, E = x.shape
    s = plain_scores(x, score)
    b = None if bias is None else np.asarray(bias, np.float64)
    none = (x == -np.inf) if b is None else (x == -np.inf) | (b == -np.inf)
    with np.errstate(all="ignore"):
        key = x.copy() if b is None else s + b
        by = key if b is not None or group_top == 1 else s
        key, by = np.where(none, -np.inf, key), np.where(none, -np.inf, by)
    ids, w = np.full((T, k), -1, np.int64), np.zeros((T, k))
    for t in range(T):
        row = key[t]
        if groups > 1:
            size = E // groups
            value = []
            for g in range(groups):
                top = in_order(by[t, g * size:(g + 1) * size], group_top)
                value.append(sum(by[t, g * size + i] for i in top) if top else -np.inf)
            kept = in_order(value, top_groups)
            row = np.where(np.isin(np.arange(E) // size, kept), row, -np.inf)
        at = in_order(row, k)
        ids[t, :len(at)] = at
        v = s[t, at]
        if renormalize and score == "softmax" and len(at) and not np.isnan(v).any():
            v = np.exp(x[t, at] - x[t, at].max())
            v = v / v.sum()
        elif renormalize:
            v = v / (v.sum() + 1e-20)
        w[t, :len(at)] = scale * v
    return ids, w, s


def span(x):
    """Range of a row's finite logits."""
    on = np.isfinite(x)
    top, low = np.where(on, x, -np.inf).max(1, keepdims=True), np.where(on, x, np.inf).min(1, keepdims=True)
    return np.where(on.any(1, keepdims=True), top - low, 0.0)


def check_route(logits, ids, weights, how):
    x = logits.double().cpu().numpy()
    want, w, _ = plain_route(x, **how)
    np.testing.assert_array_equal(ids.cpu().numpy(), want)
    got = weights.double().cpu().numpy()
    tol = (40 + 2 * how["k"] + span(x)) * U32 * np.abs(w) + 2.0 ** -126
    assert (np.isnan(got) == np.isnan(w)).all()
    assert (np.abs(got - w) <= tol)[~np.isnan(w)].all()


def make(cuda, T, E, dt, seed=0, wide=1.0):
    import torch
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    return (wide * torch.randn(T, E, device=cuda, generator=g)).to(dt)


CASES = [(1, 1, 1, 1, 1), (3, 2, 2, 1, 1), (40, 7, 3, 1, 1), (33, 8, 2, 1, 1), (100, 16, 4, 4, 2), (65, 17, 17, 1, 1),
         (30, 60, 6, 4, 2), (129, 64, 6, 8, 3), (17, 64, 64, 1, 1), (50, 128, 8, 16, 5), (21, 160, 8, 8, 3),
         (70, 256, 8, 8, 4), (9, 256, 64, 256, 200), (9, 255, 5, 85, 7), (5, 250, 9, 2, 1)]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
@pytest.mark.parametrize("T,E,k,groups,top", CASES)
def test_route(cuda, T, E, k, groups, top, dt, score):
    import torch
    from aethermoe_b200 import routing
    x = make(cuda, T, E, getattr(torch, dt), seed=T + E)
    bias = 0.1 * torch.randn(E, device=cuda)
    for b in (None, bias, 30 * bias):
        for group_top in (1, 2):
            for renorm, scale in ((False, 1.0), (True, 2.5)):
                how = dict(k=k, score=score, groups=groups, top_groups=top, group_top=group_top, renormalize=renorm,
                           scale=scale)
                ids, w = routing.route_tokens(x, bias=b, **how)
                check_route(x, ids, w, dict(how, bias=None if b is None else b.cpu().numpy()))


@pytest.mark.parametrize("E,k,groups,top", [(64, 6, 1, 1), (256, 8, 8, 4), (60, 4, 4, 2)])
def test_bias_and_logits_at_any_address(cuda, E, k, groups, top):
    """Vectors are loaded where addresses and strides allow it: the same results."""
    import torch
    from aethermoe_b200 import routing
    x, bias = make(cuda, 70, E, torch.float32, seed=E), 0.1 * torch.randn(E, device=cuda)
    how = dict(score="sigmoid", groups=groups, top_groups=top, group_top=2, renormalize=True)
    ids, w = routing.route_tokens(x, k, bias=bias, **how)
    for off in (1, 2, 4):
        b = torch.zeros(E + off, device=cuda)[off:].copy_(bias)
        y = torch.zeros(70, E + off, device=cuda)[:, off:].copy_(x)
        for xx, bb in ((x, b), (y, bias), (y, b)):
            got = routing.route_tokens(xx, k, bias=bb, **how)
            assert torch.equal(got[0], ids) and torch.equal(got[1], w), off


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_near_and_equal_keys(cuda, score):
    """Keys that float32 cannot tell apart are ordered as 64 bits order them, and
    equal ones by their index: logits on a coarse grid with biases that nearly undo
    them, groups of equal values, rows of one value."""
    import torch
    from aethermoe_b200 import routing
    E, T = 64, 200
    x = torch.randint(-3, 4, (T, E), device=cuda).float()
    s = torch.from_numpy(plain_scores(x.double().cpu().numpy(), score))
    for b in (-s[0].float(), torch.zeros(E), 0.5 - s[1].float(), torch.full((E,), 0.3)):
        b = b.to(cuda)
        for groups, top, group_top in ((1, 1, 1), (8, 3, 2), (16, 4, 1)):
            how = dict(k=8, score=score, groups=groups, top_groups=top, group_top=group_top)
            ids, w = routing.route_tokens(x, bias=b, **how)
            check_route(x, ids, w, dict(how, bias=b.cpu().numpy()))
    x = torch.full((5, E), 0.7, device=cuda).bfloat16()
    ids, w = routing.route_tokens(x, 8, score=score)
    assert (ids.cpu() == torch.arange(8)).all()
    ids, w = routing.route_tokens(x, 4, score=score, groups=8, top_groups=2, group_top=2)
    assert (ids.cpu() == torch.arange(4)).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [False, True])
def test_masked_and_special_logits(cuda, score, renorm):
    """-inf logits and biases are never chosen, rows without any choice get -1 and
    zero; the type's lowest value, infinities and NaN; both zeros are one value."""
    import torch
    from aethermoe_b200 import routing
    for dt in (torch.float32, torch.bfloat16):
        low = torch.finfo(dt).min
        for E in (8, 24, 64, 256):
            x = make(cuda, 12, E, dt, seed=E)
            x[0] = -np.inf
            x[1, 3:] = -np.inf
            x[2] = low
            x[3, 1:] = low
            x[4, ::2] = -np.inf
            x[5] = 0.0
            x[5, 1::2] = -0.0
            x[6, 5] = np.nan
            x[7, 4] = np.nan
            x[7, 6] = np.nan
            x[8] = -80.0 - torch.arange(E, device=cuda) % 4
            x[9] = 80.0
            if score == "sigmoid":
                x[10, 2] = np.inf
            bias = 0.1 * torch.randn(E, device=cuda)
            bias[1] = -np.inf
            for b in (None, bias):
                for groups, top, gt in ((1, 1, 1), (4, 2, 2), (4, 2, 1)):
                    how = dict(k=2, score=score, groups=groups, top_groups=top, group_top=gt, renormalize=renorm)
                    ids, w = routing.route_tokens(x, bias=b, **how)
                    check_route(x, ids, w, dict(how, bias=None if b is None else b.cpu().numpy()))


def test_fewer_experts_than_slots(cuda):
    import torch
    from aethermoe_b200 import dispatch as D
    from aethermoe_b200 import routing
    x = make(cuda, 50, 16, torch.float32)
    x[torch.rand(50, 16, device=cuda) < 0.8] = -np.inf
    ids, w = routing.route_tokens(x, 6, renormalize=True)
    n = (x != -np.inf).sum(1).clamp(max=6)
    assert torch.equal((ids >= 0).sum(1), n) and (w[ids < 0] == 0).all()
    rows, order = D.dispatch(torch.ones(50, 8, device=cuda), ids, 16)
    assert order.starts[-1] == n.sum()
    out = D.combine(rows, w, order)
    assert torch.allclose(out[:, 0], (n > 0).float(), atol=1e-6)


# ------------------------------------------------------------------ gradient
def plain_grad(x, ids, g, score, renorm, scale):
    """(gradient, magnitudes of its terms) in 64 bits."""
    T, E = x.shape
    s = plain_scores(x, score)
    gx, mag = np.zeros((T, E)), np.zeros((T, E))
    for t in range(T):
        at = [(j, i) for j, i in enumerate(ids[t]) if i >= 0]
        if not at:
            continue
        j, i = np.array([a[0] for a in at]), np.array([a[1] for a in at])
        gj = scale * g[t, j]
        if score == "softmax" and not renorm:
            gx[t] = -s[t] * (gj * s[t, i]).sum()
            mag[t] = s[t] * (np.abs(gj) * s[t, i]).sum()
            np.add.at(gx[t], i, s[t, i] * gj)
            np.add.at(mag[t], i, s[t, i] * np.abs(gj))
            continue
        if score == "softmax":
            q = np.exp(x[t, i] - x[t, i].max())
            q /= q.sum()
            d, m = q * (gj - (gj * q).sum()), q * (np.abs(gj) + (np.abs(gj) * q).sum())
        else:
            slope = s[t, i] / (1 + np.exp(x[t, i]))
            d, m = gj * slope, np.abs(gj) * slope
            if renorm:
                D = s[t, i].sum() + 1e-20
                d = (gj - (gj * s[t, i]).sum() / D) / D * slope
                m = (np.abs(gj) + (np.abs(gj) * s[t, i]).sum() / D) / D * slope
        np.add.at(gx[t], i, d)
        np.add.at(mag[t], i, m)
    return gx, mag


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (3, 5, 2), (40, 8, 8), (65, 17, 3), (33, 64, 6), (20, 128, 64),
                                   (50, 256, 8), (6, 250, 7)])
def test_gradient(cuda, T, E, k, dt, renorm, score):
    import torch
    from aethermoe_b200 import routing
    dt = getattr(torch, dt)
    x = make(cuda, T, E, dt, seed=E + k, wide=2.0)
    ids = torch.stack([torch.randperm(E, device=cuda)[:k] for _ in range(T)]).int()
    ids[torch.rand(T, k, device=cuda) < 0.1] = -1
    ids[0] = -1 if T > 1 else ids[0]
    if k > 1:
        ids[-1, 1] = ids[-1, 0]  # the same expert twice
    g = torch.randn(T, k, device=cuda)
    g[ids < 0] = np.nan  # of no effect
    how = dict(score=score, renormalize=renorm, scale=2.5)
    got = routing.route_tokens_backward(g, x, ids, **how)
    assert got.dtype == dt
    ref, mag = plain_grad(x.double().cpu().numpy(), ids.cpu().numpy(), g.double().cpu().numpy(), score, renorm, 2.5)
    tol = (2 * (40 + 2 * k + span(x.double().cpu().numpy())) + k) * U32 * mag + 2.0 ** -126
    if dt == torch.bfloat16:
        tol = tol + HALF_BF16 * (np.abs(ref) + tol)
    assert (np.abs(got.double().cpu().numpy() - ref) <= tol).all()
    # strided views give the same bits
    wide = torch.full((T, E + 3), 5.0, device=cuda, dtype=dt)
    out = routing.route_tokens_backward(torch.cat([g, g], 1)[:, :k], torch.cat([x, x], 1)[:, :E],
                                        torch.cat([ids, ids], 1)[:, :k], out=wide[:, :E], **how)
    assert torch.equal(out, got) and (wide[:, E:] == 5).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [False, True])
def test_gradient_against_differences(score, renorm):
    """The formula itself: central differences of the 64-bit weights."""
    rng = np.random.default_rng(3)
    x = rng.normal(size=(4, 9))
    how = dict(k=4, score=score, renormalize=renorm, scale=1.5)
    ids, w, _ = plain_route(x, **how)
    g = rng.normal(size=w.shape)
    ref, _ = plain_grad(x, ids, g, score, renorm, 1.5)
    h = 1e-5
    for e in range(9):
        d = np.zeros_like(x)
        d[:, e] = h
        (i1, w1, _), (i2, w2, _) = plain_route(x + d, **how), plain_route(x - d, **how)
        assert (i1 == ids).all() and (i2 == ids).all()
        # the third derivative is under 10 here, so the difference is within 10 h^2 and rounding
        np.testing.assert_allclose(((w1 - w2) * g).sum(1) / (2 * h), ref[:, e], atol=1e-8)


def test_autograd(cuda):
    import torch
    from aethermoe_b200 import routing
    x = make(cuda, 300, 64, torch.float32).requires_grad_()
    bias = 0.1 * torch.randn(64, device=cuda)
    how = dict(score="sigmoid", renormalize=True, scale=2.0)
    ids, w = routing.route_tokens(x, 6, bias=bias, groups=8, top_groups=3, group_top=2, **how)
    assert not ids.requires_grad and w.requires_grad
    g = torch.randn_like(w)
    w.backward(g)
    assert torch.equal(x.grad, routing.route_tokens_backward(g, x.detach(), ids, **how))
    with pytest.raises(RuntimeError, match="no gradient"):
        routing.route_tokens(x, 6, bias=bias.clone().requires_grad_())
    ids, w = routing.route_tokens(x, 6)
    (w.sum() * 0 + x.sum()).backward()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    x.grad = None
    ids, w = routing.route_tokens(x, 6, stream=s)
    torch.cuda.current_stream().wait_stream(s)
    w.backward(g)
    torch.cuda.synchronize()
    assert torch.equal(x.grad, routing.route_tokens_backward(g, x.detach(), ids))
    with pytest.raises(ValueError, match="overlaps"):
        routing.route_tokens_backward(g, x.detach(), ids, out=x.detach())


def test_captured(cuda):
    """Forward and backward captured, replayed on other values; the differentiable
    form refuses."""
    import torch
    from aethermoe_b200 import routing
    x = make(cuda, 500, 256, torch.bfloat16, seed=1)
    g = torch.randn(500, 8, device=cuda)
    bias = 0.05 * torch.randn(256, device=cuda)

    def step():
        ids, w = routing.route_tokens(x, 8, score="sigmoid", bias=bias, groups=8, top_groups=4, group_top=2)
        return ids, w, routing.route_tokens_backward(g, x, ids, score="sigmoid")
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
        leaf = x.detach().clone().requires_grad_()
        with pytest.raises(RuntimeError, match="captured"):
            routing.route_tokens(leaf, 8)
    x.copy_(make(cuda, 500, 256, torch.bfloat16, seed=2))
    graph.replay()
    for a, b in zip(got, step()):
        assert torch.equal(a, b)


def test_ids_past_the_experts_are_reported(cuda):
    import torch
    from aethermoe_b200 import _lib, routing
    x = make(cuda, 4, 8, torch.float32)
    ids = torch.tensor([[0, 8], [1, 2], [-1, 300], [7, 6]], device=cuda, dtype=torch.int32)
    g = torch.ones(4, 2, device=cuda)
    got = routing.route_tokens_backward(g, x, ids)
    assert _lib.lib().aem_device_status(None) == _lib.AEM_EDEVICE
    clean = torch.where(ids >= 8, -1, ids)
    assert torch.equal(got, routing.route_tokens_backward(g, x, clean))
    assert _lib.lib().aem_device_status(None) == _lib.AEM_OK


def test_empty_batch_and_many_rows(cuda):
    import torch
    from aethermoe_b200 import routing
    ids, w = routing.route_tokens(torch.empty(0, 8, device=cuda), 2)
    assert ids.shape == w.shape == (0, 2)
    assert routing.route_tokens_backward(w, torch.empty(0, 8, device=cuda), ids).shape == (0, 8)
    x = torch.zeros(300001, 8, device=cuda)
    x[:, 5] = 1.0
    ids, w = routing.route_tokens(x, 1)
    assert (ids == 5).all() and ids.shape == (300001, 1)
