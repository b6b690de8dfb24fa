"""Token dispatch and combine with their gradients on the GPU, against a plain
implementation in 64 bits.

Tolerances.  Orders and copied rows are exact.  A float32 sum of k products by
fused multiply-adds rounds k times: k * 2^-24 * sum |w x|.  A dot product over
d adds every term through at most d/32 + 24 roundings (a lane's chain, the
warp's tree, the block's sum).  A bf16 result adds 2^-8 of its value.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U32, HALF_BF16 = 2.0 ** -24, 2.0 ** -8


def make_ids(rng, T, k, E, masked):
    ids = np.argsort(rng.normal(size=(T, E)) - 1.1 * np.log(np.arange(1, E + 1)) * -1.0, axis=1)[:, :k]
    ids = ids.astype(np.int32)
    if masked == "some":
        ids[rng.random(ids.shape) < 0.3] = -1
        ids[T - T // 4:] = -5
    elif masked == "all":
        ids[:] = -1
    return ids


def plain_order(ids, E):
    flat = ids.reshape(-1)
    units = np.concatenate([np.flatnonzero(flat == e) for e in range(E)])
    row_of = np.full(flat.size, -1, np.int64)
    row_of[units] = np.arange(units.size)
    unit_of = np.full(flat.size, -1, np.int64)
    unit_of[:units.size] = units
    starts = np.concatenate([[0], np.cumsum([np.sum(flat == e) for e in range(E)])])
    return starts, row_of.reshape(ids.shape), unit_of


def rnd(x, dt):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x)).to(torch.float32).to(dt)


def check(got, ref, tol):
    got = got.double().cpu().numpy()
    assert got.shape == ref.shape
    bad = ~(np.abs(got - ref) <= tol)
    assert not bad.any(), (np.abs(got - ref)[bad][:4], np.broadcast_to(tol, ref.shape)[bad][:4])


SHAPES = [(1, 1, 1, 1), (1, 2, 8, 64), (3, 2, 4, 7), (37, 5, 17, 33), (128, 8, 16, 96), (129, 8, 16, 40),
          (512, 2, 256, 8), (1000, 3, 256, 24), (2500, 6, 64, 136), (700, 64, 64, 16), (33, 1, 1, 2050),
          (5000, 1, 3, 12)]


@pytest.mark.parametrize("masked", ["none", "some", "all"])
@pytest.mark.parametrize("T,k,E,d", SHAPES)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_dispatch(cuda, T, k, E, d, dtype, masked):
    import torch
    from aethermoe_b200 import dispatch as D
    rng = np.random.default_rng(T * 7 + k)
    ids = make_ids(rng, T, k, E, masked)
    x = rnd(rng.normal(size=(T, d)), getattr(torch, dtype)).to(cuda)
    starts, row_of, unit_of = plain_order(ids, E)
    rows, order = D.dispatch(x, torch.from_numpy(ids).to(cuda), E)
    np.testing.assert_array_equal(order.starts.cpu().numpy(), starts)
    np.testing.assert_array_equal(order.row_of.cpu().numpy(), row_of)
    np.testing.assert_array_equal(order.unit_of.cpu().numpy(), unit_of)
    want = np.zeros((T * k, d))
    n = starts[-1]
    want[:n] = x.double().cpu().numpy()[unit_of[:n] // k]
    np.testing.assert_array_equal(rows.double().cpu().numpy(), want)
    np.testing.assert_array_equal(D.dispatch_rows(x, order).double().cpu().numpy(), want)
    only = D.sort_tokens(torch.from_numpy(ids).to(cuda), E)
    assert torch.equal(only.row_of, order.row_of) and torch.equal(only.unit_of, order.unit_of)
    assert torch.equal(only.starts, order.starts)


@pytest.mark.parametrize("masked", ["none", "some", "all"])
@pytest.mark.parametrize("T,k,E,d", SHAPES)
@pytest.mark.parametrize("rdt,odt", [("float32", "float32"), ("bfloat16", "bfloat16"),
                                     ("float32", "bfloat16"), ("bfloat16", "float32")])
def test_combine_and_gradients(cuda, T, k, E, d, rdt, odt, masked):
    import torch
    from aethermoe_b200 import dispatch as D
    rng = np.random.default_rng(T * 5 + k + d)
    rdt, odt = getattr(torch, rdt), getattr(torch, odt)
    ids = make_ids(rng, T, k, E, masked)
    starts, row_of, unit_of = plain_order(ids, E)
    n = starts[-1]
    order = D.sort_tokens(torch.from_numpy(ids).to(cuda), E)
    w = rng.random((T, k)).astype(np.float32)
    w[row_of < 0] = np.nan  # the weight of a unit without an expert is not read
    rows = rnd(rng.normal(size=(T * k, d)), rdt).to(cuda)
    rows[n:] = float("nan")  # nor are the rows that no unit has
    go = rnd(rng.normal(size=(T, d)), odt).to(cuda)
    wt = torch.from_numpy(w).to(cuda)
    r64, g64 = rows.double().cpu().numpy(), go.double().cpu().numpy()
    live = row_of >= 0
    pick = np.where(live[:, :, None], r64[np.maximum(row_of, 0)], 0.0)  # [T, k, d]
    w64 = np.where(live, w.astype(np.float64), 0.0)

    def store(ref, tol, dt):
        return tol + (HALF_BF16 * (np.abs(ref) + tol) if dt == torch.bfloat16 else 0.0)

    ref = (pick * w64[:, :, None]).sum(1)
    tol = k * U32 * (np.abs(pick) * w64[:, :, None]).sum(1)
    check(D.combine(rows, wt, order, out_dtype=odt), ref, store(ref, tol, odt))
    ref = pick.sum(1)
    check(D.dispatch_backward(rows, order, out_dtype=odt), ref, store(ref, k * U32 * np.abs(pick).sum(1), odt))

    gr, gw = D.combine_backward(go, rows, wt, order)
    assert gr.dtype == rdt and gw.dtype == torch.float32
    ref = np.zeros((T * k, d))
    u = unit_of[:n]
    ref[:n] = w64.reshape(-1)[u][:, None] * g64[u // k]
    check(gr, ref, store(ref, U32 * np.abs(ref), rdt))
    ref = np.einsum("tkd,td->tk", pick, g64)
    check(gw, ref, (d / 32 + 24) * U32 * np.einsum("tkd,td->tk", np.abs(pick), np.abs(g64)))


def test_ids_of_any_stride(cuda):
    import torch
    from aethermoe_b200 import dispatch as D
    rng = np.random.default_rng(3)
    for T in (40, 1200):
        full = torch.from_numpy(make_ids(rng, T, 4, 9, "some")).to(cuda)
        x = torch.randn(T, 48, device=cuda)
        for ids in (full[:, :3], full.t().contiguous().t(), full[:, ::2], full[::3], full[:1].expand(T, 4)):
            xs = x[:ids.shape[0]]
            rows, order = D.dispatch(xs, ids, 9)
            want, worder = D.dispatch(xs, ids.contiguous(), 9)
            assert torch.equal(rows, want) and torch.equal(order.row_of, worder.row_of)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_rows_of_any_stride_and_alignment(cuda, dtype):
    import torch
    from aethermoe_b200 import dispatch as D
    dt = getattr(torch, dtype)
    rng = np.random.default_rng(4)
    T, k, E = 300, 3, 8
    ids = torch.from_numpy(make_ids(rng, T, k, E, "some")).to(cuda)
    order = D.sort_tokens(ids, E)
    w = torch.rand(T, k + 2, device=cuda)
    for off, d, pad in ((0, 64, 8), (1, 64, 0), (4, 20, 4), (3, 33, 7), (8, 8, 8)):
        big = torch.randn(T, off + d + pad, device=cuda).to(dt)
        x = big[:, off:off + d]
        want = D.dispatch(x.contiguous(), ids, E)[0]
        assert torch.equal(D.dispatch(x, ids, E)[0], want)
        buf = torch.full((T * k, off + d + pad), 7.0, device=cuda).to(dt)
        out = buf[:, off:off + d]
        D.dispatch(x, ids, E, out=out)
        assert torch.equal(out, want)
        assert (buf[:, :off] == 7).all() and (buf[:, off + d:] == 7).all()
        ww = w[:, 1:1 + k]
        y = D.combine(want, ww.contiguous(), order)
        assert torch.equal(D.combine(out, ww, order), y)
        obuf = torch.full((T, off + d + pad), 7.0, device=cuda).to(dt)
        D.combine(out, ww, order, out=obuf[:, off:off + d])
        assert torch.equal(obuf[:, off:off + d], y) and (obuf[:, off + d:] == 7).all()
        a = D.combine_backward(x, out, ww, order)
        b = D.combine_backward(x.contiguous(), want, ww.contiguous(), order)
        # the vector and the element form add the dot product in another order
        assert torch.equal(a[0], b[0])
        bound = (d / 32 + 24) * 2 * U32 * (want.float().abs()[order.row_of.clamp(min=0).long()] *
                                           x.float().abs()[:, None]).sum(2)
        assert ((a[1] - b[1]).abs() <= bound).all()
    # broadcast inputs: one row for every token, and a column-major one
    x = torch.randn(1, 40, device=cuda).to(dt).expand(T, 40)
    assert torch.equal(D.dispatch(x, ids, E)[0], D.dispatch(x.contiguous(), ids, E)[0])
    x = torch.randn(40, T, device=cuda).to(dt).t()
    assert torch.equal(D.dispatch(x, ids, E)[0], D.dispatch(x.contiguous(), ids, E)[0])


def test_expert_out_of_range_is_reported(cuda):
    import torch
    from aethermoe_b200 import _lib
    from aethermoe_b200 import dispatch as D
    for T in (10, 2000):
        ids = torch.zeros(T, 2, dtype=torch.int32, device=cuda)
        ids[3, 1] = 4
        ids[5, 0] = 2 ** 31 - 1
        rows, order = D.dispatch(torch.ones(T, 8, device=cuda), ids, 4)
        assert _lib.lib().aem_device_status(None) == _lib.AEM_EDEVICE
        assert "expert id" in _lib.last_error()
        assert order.row_of[3, 1] == -1 and order.row_of[5, 0] == -1 and order.starts[-1] == 2 * T - 2
        assert (rows[2 * T - 2:] == 0).all()
        assert _lib.lib().aem_device_status(None) == _lib.AEM_OK


def test_order_past_its_units_is_skipped_and_reported(cuda):
    import torch
    from aethermoe_b200 import _lib
    from aethermoe_b200 import dispatch as D
    T, k, d = 6, 2, 16
    row_of = torch.arange(T * k, dtype=torch.int32, device=cuda).reshape(T, k).contiguous()
    row_of[2, 1] = T * k
    row_of[4, 0] = 2 ** 31 - 1
    starts = torch.tensor([0, T * k], dtype=torch.int32, device=cuda)
    order = D.TokenOrder(starts, row_of, torch.zeros(T * k, dtype=torch.int32, device=cuda))
    rows = torch.randn(T * k, d, device=cuda)
    w = torch.rand(T, k, device=cuda)
    live = (row_of < T * k)[:, :, None]
    pick = torch.where(live, rows[row_of.clamp(max=T * k - 1).long()], 0.0)
    for call in (lambda: D.combine(rows, w, order), lambda: D.dispatch_rows(rows[:T], order),
                 lambda: D.combine_backward(rows[:T], rows, w, order)):
        out = call()
        assert _lib.lib().aem_device_status(None) == _lib.AEM_EDEVICE
        assert "token order" in _lib.last_error()
    assert out[1][2, 1] == 0 and out[1][4, 0] == 0
    torch.testing.assert_close(D.combine(rows, w, order), (pick * w[:, :, None]).sum(1))
    assert _lib.lib().aem_device_status(None) == _lib.AEM_EDEVICE


def test_empty_batch(cuda):
    import torch
    from aethermoe_b200 import dispatch as D
    x = torch.zeros(0, 16, device=cuda)
    rows, order = D.dispatch(x, torch.zeros(0, 2, dtype=torch.int32, device=cuda), 4)
    assert rows.shape == (0, 16) and order.starts.tolist() == [0] * 5
    w = torch.zeros(0, 2, device=cuda)
    assert D.combine(rows, w, order).shape == (0, 16)
    gr, gw = D.combine_backward(x, rows, w, order)
    assert gr.shape == (0, 16) and gw.shape == (0, 2)


def test_infinities_stay_with_their_rows(cuda):
    import torch
    from aethermoe_b200 import dispatch as D
    T, k, E, d = 50, 2, 4, 24
    rng = np.random.default_rng(9)
    ids = torch.from_numpy(make_ids(rng, T, k, E, "none")).to(cuda)
    x = torch.randn(T, d, device=cuda)
    x[7, 3], x[8, 4], x[9, 5] = float("inf"), float("nan"), -float("inf")
    rows, order = D.dispatch(x, ids, E)
    out = D.combine(rows, torch.full((T, k), 0.5, device=cuda), order)
    assert torch.equal(out.isnan(), x.isnan()) and torch.equal(out.isinf(), x.isinf())


def test_autograd_against_differences(cuda):
    """Whole numbers small enough that every float32 sum is exact, so a central
    difference of the bilinear layer equals its gradient bit for bit."""
    import torch
    from aethermoe_b200 import dispatch as D
    rng = np.random.default_rng(11)
    for T, k, E, d in ((9, 2, 4, 10), (600, 3, 16, 8)):
        ids = torch.from_numpy(make_ids(rng, T, k, E, "some")).to(cuda)
        scale = torch.from_numpy(rng.integers(-3, 4, size=(E, d)).astype(np.float32)).to(cuda)
        c = torch.from_numpy(rng.integers(-3, 4, size=(T, d)).astype(np.float32)).to(cuda)
        x = torch.from_numpy(rng.integers(-4, 5, size=(T, d)).astype(np.float32)).to(cuda)
        w = torch.from_numpy(rng.integers(-4, 5, size=(T, k)).astype(np.float32)).to(cuda)

        def loss(x, w):
            rows, order = D.dispatch(x, ids, E)
            e = (torch.arange(T * k, device=cuda)[:, None] >= order.starts[None, 1:E]).sum(1)
            return (D.combine(rows * scale[e], w, order).double() * c).sum()

        xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
        loss(xg, wg).backward()
        for i in range(12):
            dx = torch.zeros_like(x)
            dx[rng.integers(T), rng.integers(d)] = 1.0
            dw = torch.zeros_like(w)
            dw[rng.integers(T), rng.integers(k)] = 1.0
            assert (loss(x + dx, w) - loss(x - dx, w)) / 2 == (xg.grad * dx).sum()
            assert (loss(x, w + dw) - loss(x, w - dw)) / 2 == (wg.grad * dw).sum()


def test_autograd_of_shared_and_broadcast_inputs(cuda):
    import torch
    from aethermoe_b200 import dispatch as D
    rng = np.random.default_rng(12)
    T, k, E, d = 200, 2, 8, 32
    ids = torch.from_numpy(make_ids(rng, T, k, E, "none")).to(cuda)
    one = torch.ones(1, d, device=cuda, requires_grad=True)
    w = torch.ones(1, k, device=cuda, requires_grad=True)
    rows, order = D.dispatch(one.expand(T, d), ids, E)
    again = D.dispatch_rows(one.expand(T, d), order)
    D.combine(rows + again, w.expand(T, k), order).sum().backward()  # a gradient of stride 0
    assert (one.grad == 2 * T * k).all() and (w.grad == 2 * T * d).all()
    # no gradient asked for: none is made
    x = torch.randn(T, d, device=cuda)
    out = D.combine(D.dispatch(x, ids, E)[0], w.expand(T, k), order)
    out.sum().backward()
    assert x.grad is None
    with pytest.raises(RuntimeError, match="out="):
        D.dispatch(one.expand(T, d), ids, E, out=torch.empty(T * k, d, device=cuda))


def test_differentiable_form_refuses_capture(cuda):
    import torch
    from aethermoe_b200 import dispatch as D
    x = torch.ones(4, 8, device=cuda, requires_grad=True)
    ids = torch.zeros(4, 1, dtype=torch.int32, device=cuda)
    eager, order = D.dispatch(x, ids, 2)  # lives through the capture
    g = torch.cuda.CUDAGraph()
    said = []
    with torch.cuda.graph(g):
        y = torch.zeros(4, device=cuda) + 1
        for call in (lambda: D.dispatch(x, ids, 2), lambda: D.dispatch_rows(x, order),
                     lambda: D.combine(eager, torch.ones(4, 1, device=cuda), order)):
            try:
                call()
            except RuntimeError as e:
                said.append("captured" in str(e))
        gx = D.dispatch_backward(eager.detach(), order)
    g.replay()
    torch.cuda.synchronize()
    assert said == [True] * 3 and (gx == 1).all() and (y == 1).all()
    eager.sum().backward()
    assert (x.grad == 1).all()


def test_captured_and_replayed(cuda):
    """Two graphs of the whole step, replayed in turn on new inputs."""
    import torch
    from aethermoe_b200 import dispatch as D
    rng = np.random.default_rng(13)
    graphs = []
    for T, k, E, d in ((64, 2, 8, 64), (3000, 4, 32, 40)):
        x = torch.randn(T, d, device=cuda)
        ids = torch.from_numpy(make_ids(rng, T, k, E, "some")).to(cuda)
        w = torch.rand(T, k, device=cuda)

        def step(x=x, ids=ids, w=w, E=E):
            rows, order = D.dispatch(x, ids, E)
            out = D.combine(rows, w, order)
            gr, gw = D.combine_backward(out, rows, w, order)
            return rows, order.starts, order.row_of, out, gr, gw, D.dispatch_backward(gr, order)

        step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = step()
        graphs.append((g, got, step, x, ids, w, (T, k, E)))
    for it in range(3):
        for g, got, step, x, ids, w, (T, k, E) in graphs:
            x.normal_()
            w.uniform_()
            ids.copy_(torch.from_numpy(make_ids(rng, T, k, E, "some")))
            g.replay()
        for g, got, step, *_ in graphs:
            for a, b in zip(got, step()):
                assert torch.equal(a, b)


def test_other_stream_and_repeats(cuda):
    import torch
    from aethermoe_b200 import dispatch as D
    rng = np.random.default_rng(14)
    T, k, E, d = 2000, 3, 16, 72
    ids = torch.from_numpy(make_ids(rng, T, k, E, "some")).to(cuda)
    x = torch.randn(T, d, device=cuda)
    w = torch.rand(T, k, device=cuda)
    rows, order = D.dispatch(x, ids, E)
    out = D.combine(rows, w, order)
    gr, gw = D.combine_backward(out, rows, w, order)
    side = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in side:  # two at once
        s.wait_stream(torch.cuda.current_stream())
        r, o = D.dispatch(x, ids, E, stream=s)
        y = D.combine(r, w, o, stream=s)
        got.append((r, y) + tuple(D.combine_backward(y, r, w, o, stream=s)))
    for s in side:
        torch.cuda.current_stream().wait_stream(s)
    for g in got:
        for a, b in zip(g, (rows, out, gr, gw)):
            assert torch.equal(a, b)


def test_past_32_bit_offsets(cuda):
    """4.9 GB of rows: element offsets past 2^31."""
    import torch
    from aethermoe_b200 import dispatch as D
    T, k, E, d = 150001, 2, 4, 8192
    ids = torch.randint(0, 4, (T, 1), device=cuda, dtype=torch.int32)
    ids = torch.cat([ids, (ids + 1) % 4], 1)
    x = torch.randint(-8, 9, (T, d), device=cuda, dtype=torch.int8).to(torch.bfloat16)
    rows, order = D.dispatch(x, ids, E)
    at = torch.randint(0, T * k, (500,), device=cuda)
    at[:2] = torch.tensor([0, T * k - 1])
    assert torch.equal(rows[at], x[order.unit_of[at].long() // k])
    w = torch.full((T, k), 0.5, device=cuda)
    assert torch.equal(D.combine(rows, w, order), x)
    gr, gw = D.combine_backward(x, rows, w, order)
    assert torch.equal(gr[at] * 2, rows[at])
    t = torch.randint(0, T, (300,), device=cuda)
    t[0] = T - 1
    assert torch.equal(gw[t, 1].double(), (x[t].double() ** 2).sum(1))
