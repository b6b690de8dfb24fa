"""Calls of the dispatch, combine and 4-bit products that their documentation
allows and that lie away from ordinary use: rows longer than one part of a
kernel holds, non-finite values on every path, outputs with a padded row
stride, two threads at once, a whole training step.  Tolerances of the
products are derived in ``test_q4_gpu``."""
import threading

import pytest

from test_q4_gpu import check, product, weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("xdt", ["bfloat16", "float32"])
@pytest.mark.parametrize("K,M,gs", [(16501, 1, 128), (16501, 40, 64), (25001, 1, 32), (25001, 4, 128),
                                    (33000, 3, 64), (20480, 9, 32)])
def test_long_rows(cuda, K, M, gs, xdt):
    import torch
    from aethermoe_b200 import q4
    q, s = weights(cuda, 1, K, 40, gs, torch.float32, seed=K + M)
    w = q4.Q4Weight(q[0], s[0], gs)
    x = torch.randn(M, K, device=cuda).to(getattr(torch, xdt))
    ref, A = product(x, q[0], s[0], gs)
    check(q4.q4_matmul(x, w, out_dtype=torch.float32), ref, A, s.shape[1])


@pytest.mark.parametrize("xdt", ["bfloat16", "float32"])
@pytest.mark.parametrize("K", [256, 20001])
@pytest.mark.parametrize("M", [1, 2, 4, 6, 17])
def test_non_finite_values_on_every_path(cuda, M, K, xdt):
    """An infinity or NaN anywhere in a row decides that row alone, and the other
    elements of a call keep their precision; a row of zeros is zero."""
    import torch
    from aethermoe_b200 import q4
    q, s = weights(cuda, 1, K, 36, 64, torch.float32, low=1)  # no zero weight: inf stays inf
    w = q4.Q4Weight(q[0], s[0], 64)
    x = torch.randn(M, K, device=cuda).to(getattr(torch, xdt))
    for at in (0, K // 2, K - 1):
        for v in (float("inf"), -float("inf"), float("nan")):
            y = x.clone()
            y[M - 1, at] = v
            out = q4.q4_matmul(y, w, out_dtype=torch.float32)
            last = out[M - 1]
            assert last.isnan().all() if v != v else (last == v).all()
            if M > 1:
                ref, A = product(y[:M - 1], q[0], s[0], 64)
                check(out[:M - 1], ref, A, s.shape[1])
    y = x.clone()
    y[M - 1] = 0
    assert (q4.q4_matmul(y, w)[M - 1] == 0).all()


@pytest.mark.parametrize("odt", ["bfloat16", "float32"])
@pytest.mark.parametrize("M", [1, 3, 8, 33])
@pytest.mark.parametrize("N,ld", [(50, 64), (129, 136), (6, 8)])
def test_padded_output_rows(cuda, N, ld, M, odt):
    """Columns behind N belong to the caller, whatever vectors the rest allows."""
    import torch
    from aethermoe_b200 import q4
    q, s = weights(cuda, 1, 300, N, 64, torch.float32, seed=N)
    w = q4.Q4Weight(q[0], s[0], 64)
    x = torch.randn(M, 300, device=cuda)
    ref, A = product(x, q[0], s[0], 64)
    buf = torch.full((M, ld), 7.0, device=cuda, dtype=getattr(torch, odt))
    check(q4.q4_matmul(x, w, out=buf[:, :N]), ref, A, s.shape[1])
    assert (buf[:, N:] == 7).all()


def test_overlaps_and_gradients_are_refused(cuda):
    import torch
    from aethermoe_b200 import dispatch as D
    from aethermoe_b200 import q4
    q, s = weights(cuda, 1, 64, 64, 32, torch.float32)
    w = q4.Q4Weight(q[0], s[0], 32)
    buf = torch.randn(8, 192, device=cuda)
    x = buf[:, :64]
    ids = torch.zeros(8, 1, dtype=torch.int32, device=cuda)
    rows, order = D.dispatch(x, ids, 4)
    val = torch.ones(8, 1, device=cuda)
    for bad in (lambda: q4.q4_matmul(x, w, out=x), lambda: q4.q4_matmul(x, w, out=buf[:, 32:96]),
                lambda: q4.grouped_q4_matmul(x, w, torch.tensor([0, 8], dtype=torch.int32, device=cuda), out=x),
                lambda: D.dispatch(x, ids, 4, out=x), lambda: D.dispatch_rows(x, order, out=x),
                lambda: D.combine(rows, val, order, out=rows), lambda: D.dispatch_backward(rows, order, out=rows)):
        with pytest.raises(ValueError, match="overlaps"):
            bad()
    ref = q4.q4_matmul(x, w)
    assert torch.equal(q4.q4_matmul(x, w, out=buf[:, 64:128]), ref)  # columns of one buffer do not overlap
    x = x.detach().clone().requires_grad_()
    for bad in (lambda: q4.q4_matmul(x, w),
                lambda: q4.grouped_q4_matmul(x, w, torch.tensor([0, 8], dtype=torch.int32, device=cuda))):
        with pytest.raises(RuntimeError, match="no gradient"):
            bad()
    with torch.no_grad():
        assert torch.equal(q4.q4_matmul(x, w), ref)


def test_two_threads(cuda):
    """Calls from two threads, each on its own stream, share weights and nothing else."""
    import torch
    from aethermoe_b200 import dispatch as D
    from aethermoe_b200 import q4
    E, d, f = 8, 512, 256
    q, s = weights(cuda, E, d, f, 64, torch.bfloat16)
    w = q4.Q4Weight(q, s, 64)
    cases = []
    for i, T in enumerate((40, 700)):
        g = torch.Generator(device=cuda).manual_seed(i)
        x = torch.randn(T, d, device=cuda, generator=g).bfloat16()
        ids = torch.randint(-1, E, (T, 2), device=cuda, dtype=torch.int32, generator=g)
        val = torch.rand(T, 2, device=cuda, generator=g)
        cases.append((x, ids, val))

    def step(x, ids, val):
        rows, order = D.dispatch(x, ids, E)
        y = q4.grouped_q4_matmul(rows, w, order.starts, relu=True)
        return D.combine(y, val, order)
    want = [step(*c) for c in cases]
    torch.cuda.synchronize()
    got = [[], []]

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i].append(step(*cases[i]))
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(2):
        assert len(got[i]) == 20 and all(torch.equal(o, want[i]) for o in got[i])


@pytest.mark.parametrize("T,k,E", [(5, 2, 4), (300, 3, 6)])
def test_training_step(cuda, T, k, E):
    """Dispatch, experts and combine as one differentiable step, against the same
    step without any sorting in 64 bits.  On whole numbers every float32 sum is
    exact (below 2^24), so the gradients must be equal, not near."""
    import torch
    from aethermoe_b200 import dispatch as D
    d, f = 24, 16
    g = torch.Generator(device=cuda).manual_seed(T)

    def whole(*shape):
        return torch.randint(-3, 4, shape, device=cuda, generator=g).float()
    x, w, val, go = whole(T, d), whole(E, d, f), whole(T, k), whole(T, f)
    ids = torch.randint(-1, E, (T, k), device=cuda, dtype=torch.int32, generator=g)
    x, w, val = (t.requires_grad_() for t in (x, w, val))
    rows, order = D.dispatch(x, ids, E)
    bounds = order.starts.tolist()
    y = torch.cat([rows[a:b] @ w[e] for e, (a, b) in enumerate(zip(bounds, bounds[1:]))] +
                  [rows.new_zeros(T * k - bounds[E], f)])
    out = D.combine(y, val, order)
    out.backward(go)
    x2, w2, v2 = (t.detach().double().requires_grad_() for t in (x, w, val))
    on = (ids >= 0).double()
    ref = torch.einsum("td,tkdf,tk->tf", x2, w2[ids.clamp(min=0).long()], v2 * on)
    ref.backward(go.double())
    assert torch.equal(out.double(), ref)
    for a, b in ((x, x2), (w, w2), (val, v2)):
        assert torch.equal(a.grad.double(), b.grad)


@pytest.mark.parametrize("gs", [32, 64, 128])
@pytest.mark.parametrize("xdt,most", [("bfloat16", 14), ("bfloat16", 30), ("float32", 6), ("float32", 12)])
@pytest.mark.parametrize("K", [100, 384, 1300])
def test_more_tiles_than_a_wave(cuda, K, xdt, most, gs):
    """Ragged groups whose tiles are several waves of CTAs, over one, three and eleven
    blocks of K; empty groups lie first, last and between."""
    import torch
    from aethermoe_b200 import q4
    G, N = 96, 700
    q, s = weights(cuda, G, K, N, gs, torch.float32, seed=K)
    w = q4.Q4Weight(q, s, gs)
    counts = torch.randint(0, most + 1, (G,), generator=torch.Generator().manual_seed(K + most))
    counts[0] = counts[50] = counts[-1] = 0
    counts[7] = 3 * most + 1
    starts = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)])
    M = int(starts[-1]) + 5
    x = torch.randn(M, K, device=cuda).to(getattr(torch, xdt))
    buf = torch.full((M, N), 7.0, device=cuda)
    out = q4.grouped_q4_matmul(x, w, starts.int().to(cuda), out=buf)
    assert (out[M - 5:] == 7).all()
    for g in range(G):
        a, b = int(starts[g]), int(starts[g + 1])
        if a < b:
            ref, A = product(x[a:b], q[g], s[g], gs)
            check(out[a:b], ref, A, s.shape[1])
    again = q4.grouped_q4_matmul(x, w, starts.int().to(cuda), relu=True, out_dtype=torch.float32)
    assert torch.equal(again[:M - 5], out[:M - 5].clamp(min=0))


@pytest.mark.parametrize("gs", [32, 64, 128])
@pytest.mark.parametrize("xdt,M", [("bfloat16", 33), ("bfloat16", 64), ("bfloat16", 65), ("bfloat16", 150),
                                   ("float32", 32), ("float32", 33)])
@pytest.mark.parametrize("K,N", [(100, 7000), (1500, 6500), (5000, 6500)])
def test_widest_row_tiles(cuda, K, N, M, xdt, gs):
    """Enough channels that the widest row tiles are taken, with and without a split K."""
    import torch
    from aethermoe_b200 import q4
    q, s = weights(cuda, 1, K, N, gs, torch.bfloat16, seed=M)
    w = q4.Q4Weight(q[0], s[0], gs)
    x = torch.randn(M, K, device=cuda).to(getattr(torch, xdt))
    ref, A = product(x, q[0], s[0], gs)
    check(q4.q4_matmul(x, w, out_dtype=torch.float32), ref, A, s.shape[1])


def test_combine_without_weights(cuda):
    """No weights mean weights of 1, in the sum and in the gradients."""
    import torch
    from aethermoe_b200 import dispatch as D
    T, k, E, d = 40, 3, 8, 20
    ids = torch.randint(-1, E, (T, k), device=cuda, dtype=torch.int32)
    order = D.sort_tokens(ids, E)
    rows = torch.randn(T * k, d, device=cuda, requires_grad=True)
    go = torch.randn(T, d, device=cuda)
    one = torch.ones(T, k, device=cuda)
    out = D.combine(rows, None, order)
    assert torch.equal(out, D.combine(rows.detach(), one, order))
    out.backward(go)
    want, gw = D.combine_backward(go, rows.detach(), one, order)
    assert torch.equal(rows.grad, want)
    again, gw2 = D.combine_backward(go, rows.detach(), None, order)
    assert torch.equal(again, want) and torch.equal(gw2, gw)


@pytest.mark.parametrize("sdt", ["float32", "bfloat16"])
@pytest.mark.parametrize("wdt", ["float32", "bfloat16"])
@pytest.mark.parametrize("N", [33, 36])
def test_quantize_shows_non_finite_weights(cuda, N, wdt, sdt):
    import torch
    from aethermoe_b200 import q4
    wdt, sdt = getattr(torch, wdt), getattr(torch, sdt)
    w = torch.randn(200, N, device=cuda).to(wdt)
    q0, s0 = q4.quantize_q4(w, 64, sdt)
    w[70, 3], w[5, 30] = float("nan"), -float("inf")
    q, s = q4.quantize_q4(w, 64, sdt)
    assert s[1, 3].isnan() and s[0, 30] == float("inf") and (q.abs() <= 7).all()
    q[64:128, 3], s[1, 3], q[:64, 30], s[0, 30] = q0[64:128, 3], s0[1, 3], q0[:64, 30], s0[0, 30]
    assert torch.equal(q, q0) and torch.equal(s, s0)
