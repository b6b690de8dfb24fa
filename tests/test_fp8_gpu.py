"""8-bit quantisation and the products with 8-bit weights on the GPU, against a
plain implementation in 64 bits.

Quantisation is defined in float32 and equal bit for bit.  Tolerance of a product
of quantised rows with A = sum_k |xs xq ws wq|: an MMA adds 32 products to its
accumulator, each aligned to the largest with at least 24 bits, so it loses at
most 33 * 2^-23 of the magnitudes it adds, and a block is 4 MMAs: 132 * 2^-23 A.
The product of the scales rounds once, the sums over B blocks and between the
CTAs of a cluster (7) each: (B + 8) 2^-24 A.  A bf16 result adds 2^-8 of its value.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HALF_BF16 = 2.0 ** -8


def blocks(n):
    return -(-n // 128)


def plain_rows(x):
    """(q, scale) of rows in blocks of 128, by the definition, in float32."""
    import torch
    M, K = x.shape
    p = torch.nn.functional.pad(x.float(), (0, -K % 128)).reshape(M, -1, 128)
    a = p.abs().amax(2)
    s = a / torch.full_like(a, 448.0)
    s = torch.where(s < 2.0 ** -126, torch.full_like(s, 2.0 ** -126), s)
    return (p / s[:, :, None]).to(torch.float8_e4m3fn).reshape(M, -1)[:, :K], s


def value(q, s):
    return q.double() * s.double().repeat_interleave(128, -1)[..., :q.shape[-1]]


def weight_value(q, s):
    return q.double() * s.double().repeat_interleave(128, -2)[..., :q.shape[-2], :].repeat_interleave(
        128, -1)[..., :q.shape[-1]]


def check(got, x, w, B):
    import torch
    ref, A = x @ w, x.abs() @ w.abs()
    tol = (132 * 2.0 ** -23 + (B + 8) * 2.0 ** -24) * A
    if got.dtype == torch.bfloat16:
        tol = tol + HALF_BF16 * (ref.abs() + tol)
    bad = ~((got.double() - ref).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), (got.double() - ref).abs()[bad][:4], tol[bad][:4])


def weights(cuda, G, K, N, seed=0):
    import torch
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    q = (torch.randn(G, K, N, device=cuda, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    return q, torch.rand(G, blocks(K), blocks(N), device=cuda, generator=g) + 0.25


# ------------------------------------------------------------------ quantisation
@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
@pytest.mark.parametrize("M,K", [(1, 1), (3, 127), (5, 128), (7, 129), (33, 300), (64, 2048), (130, 1000), (2, 14336)])
def test_rows(cuda, M, K, dt):
    import torch
    from aethermoe_b200 import fp8
    dt = getattr(torch, dt)
    x = (torch.randn(M, K + 5, device=cuda) * torch.logspace(-12, 12, M, device=cuda)[:, None]).to(dt)
    for v in (x[:, :K], x[:, :K].contiguous(), x[:, 3:K + 3]):
        rows = fp8.quantize_fp8(v)
        q, s = plain_rows(v)
        assert rows.q.shape == (M, K) and rows.scale.shape == (M, blocks(K))
        assert torch.equal(rows.scale, s) and torch.equal(rows.q.float(), q.float())


def test_quotients_next_to_a_border(cuda):
    """Values whose quotient lies at or next to the middle of two e4m3 values, and
    scales from the smallest to the largest, where the division itself is made."""
    import torch
    from aethermoe_b200 import fp8
    e4m3 = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    middle = (e4m3[1:] + e4m3[:-1]) / 2
    for top in (448.0, 447.0, 1.0, 3.1e-3, 1e-30, 2.0 ** -83, 1.3 * 2.0 ** -81, 1e-40, 3e38, 1.7e9, 5e20):
        s = (torch.tensor(top) / torch.tensor(448.0)).clamp(min=2.0 ** -126).double()
        rows = []
        for step in range(-3, 4):
            v = (middle * s).float()
            v = (v.view(torch.int32) + step).view(torch.float32)
            row = torch.zeros(2, 128)
            row[:, 0] = top
            row[0, 1:127] = v.clamp(max=top)
            row[1, 1:127] = -v.clamp(max=top)
            rows.append(row)
        x = torch.cat(rows).to(cuda)
        got = fp8.quantize_fp8(x)
        q, s = plain_rows(x)
        assert torch.equal(got.scale, s) and torch.equal(got.q.float(), q.float()), top


def test_special_values(cuda):
    """Zeros, the smallest and largest numbers, NaN and infinities: their blocks show
    them, other blocks and rows do not."""
    import torch
    from aethermoe_b200 import fp8
    for dt in (torch.float32, torch.bfloat16):
        x = torch.randn(8, 384, device=cuda).to(dt)
        x[0] = 0
        x[1, 130] = np.nan
        x[2, 5] = np.inf
        x[3, 300] = -np.inf
        x[4] = torch.finfo(dt).max
        x[5] = torch.finfo(dt).tiny
        x[6] = 0
        x[6, 1] = 1e-45 if dt == torch.float32 else 9.2e-41
        got = fp8.quantize_fp8(x)
        q, s = plain_rows(x)
        assert torch.equal(got.scale.nan_to_num(nan=-1.0), s.nan_to_num(nan=-1.0))
        assert torch.equal(got.q.float().nan_to_num(nan=999.0), q.float().nan_to_num(nan=999.0))
        w = fp8.Fp8Weight(*fp8.quantize_fp8_weight(torch.randn(384, 64, device=cuda)))
        y = fp8.fp8_matmul(x, w, out_dtype=torch.float32)
        shows = torch.isfinite(y).all(1)
        assert shows.tolist() == [True, False, False, False, bool(shows[4]), True, True, True]
        assert not torch.isfinite(y[1:4]).any() and (y[0] == 0).all()


@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
@pytest.mark.parametrize("G,K,N", [(1, 1, 1), (2, 100, 60), (1, 128, 128), (3, 129, 257), (1, 512, 1408), (2, 300, 132)])
def test_weight_quantisation(cuda, G, K, N, dt):
    import torch
    from aethermoe_b200 import fp8
    w = torch.randn(G, K, N, device=cuda).to(getattr(torch, dt))
    w[0, 0, 0] = 30.0
    q, s = fp8.quantize_fp8_weight(w)
    assert q.shape == w.shape and s.shape == (G, blocks(K), blocks(N))
    p = torch.nn.functional.pad(w.float(), (0, -N % 128, 0, -K % 128)).reshape(G, blocks(K), 128, blocks(N), 128)
    a = p.abs().amax((2, 4))
    want = a / torch.full_like(a, 448.0)
    assert torch.equal(s, want)
    pq = (p / want[:, :, None, :, None]).to(torch.float8_e4m3fn).reshape(G, blocks(K) * 128, -1)[:, :K, :N]
    assert torch.equal(q.float(), pq.float())
    if G == 1:
        q1, s1 = fp8.quantize_fp8_weight(w[0])
        assert torch.equal(q1.float(), q[0].float()) and torch.equal(s1, s[0])


# ------------------------------------------------------------------ products
SIZES = [(1, 1, 1), (5, 7, 3), (64, 16, 1), (128, 128, 16), (100, 50, 9), (129, 130, 17), (333, 47, 33),
         (1000, 100, 65), (2048, 96, 64), (520, 600, 128), (256, 384, 129), (4096, 64, 2), (8200, 31, 7),
         (130, 1000, 260), (1024, 512, 300), (640, 520, 1030)]


@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
@pytest.mark.parametrize("K,N,M", SIZES)
def test_product_and_gradient(cuda, K, N, M, dt):
    import torch
    from aethermoe_b200 import _lib, fp8
    dt = getattr(torch, dt)
    q, s = weights(cuda, 2, K, N, seed=K + N)
    w = fp8.Fp8Weight(q, s)
    x, g = torch.randn(M, K, device=cuda).to(dt), torch.randn(M, N, device=cuda).to(dt)
    for group in range(2):
        wv = weight_value(q[group], s[group])
        for odt in (torch.float32, torch.bfloat16):
            check(fp8.fp8_matmul(x, w, group, out_dtype=odt), value(*plain_rows(x)), wv, blocks(K))
            check(fp8.fp8_matmul_backward(g, w, group, out_dtype=odt), value(*plain_rows(g)), wv.t(), blocks(N))
    assert fp8.fp8_matmul(x, w).dtype == dt
    # rows quantised before give the same bits, as given and as copies of other strides
    rows = fp8.quantize_fp8(x)
    want = fp8.fp8_matmul(x, w, out_dtype=torch.float32)
    assert torch.equal(fp8.fp8_matmul(rows, w), want)
    own = fp8.Fp8Rows(rows.q.contiguous(), rows.scale.contiguous())
    assert torch.equal(fp8.fp8_matmul(own, w), want)
    assert torch.equal(fp8.fp8_matmul(own, w), want)
    turned = fp8.Fp8Rows(rows.q.t().contiguous().t(), rows.scale.t().contiguous().t())
    assert torch.equal(fp8.fp8_matmul(turned, w), want)
    # other strides and alignments of x and out
    wide = torch.zeros(M, K + 3, device=cuda, dtype=dt)
    wide[:, 1:K + 1] = x
    out = torch.full((M, N + 3), 7.0, device=cuda)
    assert torch.equal(fp8.fp8_matmul(wide[:, 1:K + 1], w, out=out[:, 2:N + 2]), want)
    assert (out[:, :2] == 7).all() and (out[:, N + 2:] == 7).all()
    _lib.check(_lib.lib().aem_device_status(None))


def test_whole_numbers_are_exact(cuda):
    """Whole numbers and scales of one: every sum is exact, results equal bit for bit,
    in both directions and for all row tiles."""
    import torch
    from aethermoe_b200 import fp8
    for K, N in ((4096, 256), (1472, 352), (256, 2304)):
        q = torch.randint(-8, 9, (K, N), device=cuda).float()
        w = fp8.Fp8Weight(q.to(torch.float8_e4m3fn), torch.ones(blocks(K), blocks(N), device=cuda))
        for M in (1, 16, 20, 64, 100, 300, 700):
            for dt in (torch.float32, torch.bfloat16):
                x = torch.randint(-8, 9, (M, K), device=cuda).to(dt)
                x[:, ::128] = 448.0  # so the scales are one
                assert torch.equal(fp8.fp8_matmul(x, w, out_dtype=torch.float32).double(), x.double() @ q.double())
                g = torch.randint(-8, 9, (M, N), device=cuda).to(dt)
                g[:, ::128] = -448.0
                assert torch.equal(fp8.fp8_matmul_backward(g, w, out_dtype=torch.float32).double(),
                                   g.double() @ q.double().t())


def test_gradient_against_differences(cuda):
    """On whole numbers nothing rounds, so a difference of the product is its
    gradient's product exactly."""
    import torch
    from aethermoe_b200 import fp8
    K, N, M = 300, 200, 5
    q = torch.randint(-8, 9, (K, N), device=cuda).float()
    w = fp8.Fp8Weight(q.to(torch.float8_e4m3fn), torch.ones(blocks(K), blocks(N), device=cuda))
    x = torch.randint(-6, 7, (M, K), device=cuda).float()
    x[:, ::128] = 448.0
    g = torch.randint(-6, 7, (M, N), device=cuda).float()
    g[:, ::128] = 448.0
    leaf = x.clone().requires_grad_()
    fp8.fp8_matmul(leaf, w).backward(g)
    for k in (1, 77, 127, 130, 255, 299):
        d = torch.zeros_like(x)
        d[:, k] = 2.0
        diff = ((fp8.fp8_matmul(x + d, w) - fp8.fp8_matmul(x - d, w)).double() * g.double()).sum(1) / 4
        assert torch.equal(diff, leaf.grad[:, k].double())


# ------------------------------------------------------------------ grouped
COUNTS = [(1, [5]), (4, [0, 0, 0, 0]), (4, [1, 0, 17, 3]), (8, [40, 0, 64, 65, 128, 1, 0, 33]), (3, [0, 300, 0]),
          (17, [3] * 17), (64, [6] * 64), (256, [1] * 100 + [0] * 56 + [2] * 100), (5, [700, 3, 0, 260, 128])]


@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
@pytest.mark.parametrize("G,counts", COUNTS)
@pytest.mark.parametrize("K,N", [(256, 384), (200, 70)])
def test_grouped(cuda, G, counts, K, N, dt):
    import torch
    from aethermoe_b200 import _lib, fp8
    dt = getattr(torch, dt)
    q, s = weights(cuda, G, K, N, seed=G)
    w = fp8.Fp8Weight(q, s)
    first, rest = (0, 0) if sum(counts) % 2 else (3, 9)  # rows outside every group
    starts = torch.tensor(np.cumsum([first] + counts), dtype=torch.int32, device=cuda)
    M = int(starts[-1]) + rest
    if M == 0:
        return
    x, g = torch.randn(M, K, device=cuda).to(dt), torch.randn(M, N, device=cuda).to(dt)
    x[:first] = np.nan
    x[M - rest:] = np.nan
    xv, gv = value(*plain_rows(x)), value(*plain_rows(g))
    for odt in (torch.float32, torch.bfloat16):
        out = torch.full((M, N + 1), 9.0, device=cuda, dtype=odt)
        fp8.grouped_fp8_matmul(x, w, starts, out=out[:, :N])
        relu = fp8.grouped_fp8_matmul(fp8.quantize_fp8(x), w, starts, relu=True, out_dtype=odt)
        back = fp8.grouped_fp8_matmul_backward(g, w, starts, out_dtype=odt)
        for e in range(G):
            a, b = int(starts[e]), int(starts[e + 1])
            if a == b:
                continue
            wv = weight_value(q[e], s[e])
            check(out[a:b, :N], xv[a:b], wv, blocks(K))
            check(back[a:b], gv[a:b], wv.t(), blocks(N))
            assert torch.equal(relu[a:b], torch.relu(out[a:b, :N]))
        assert (out[:first] == 9).all() and (out[M - rest:] == 9).all() and (out[:, N] == 9).all()
        assert (back[:first] == 0).all() and (back[M - rest:] == 0).all()
    _lib.check(_lib.lib().aem_device_status(None))


def test_grouped_gradient(cuda):
    import torch
    from aethermoe_b200 import fp8
    q, s = weights(cuda, 4, 256, 384)
    w = fp8.Fp8Weight(q, s)
    starts = torch.tensor([0, 30, 30, 100, 130], dtype=torch.int32, device=cuda)
    x = torch.randn(140, 256, device=cuda, dtype=torch.bfloat16).requires_grad_()
    y = fp8.grouped_fp8_matmul(x, w, starts, out_dtype=torch.float32)
    assert (y[130:] == 0).all()
    g = torch.randn_like(y)
    y.backward(g)
    assert x.grad.dtype == torch.bfloat16
    assert torch.equal(x.grad, fp8.grouped_fp8_matmul_backward(g, w, starts, out_dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="relu"):
        fp8.grouped_fp8_matmul(x, w, starts, relu=True)
    y = fp8.grouped_fp8_matmul(x, w, starts)
    starts.add_(0)  # written since
    with pytest.raises(RuntimeError, match="modified"):
        y.backward(torch.randn_like(y))


def test_large_groups_of_many_experts(cuda):
    """Groups of hundreds of rows, none a multiple of a tile."""
    import torch
    from aethermoe_b200 import fp8
    counts = [531, 0, 255, 257, 1, 513, 128, 700]
    q, s = weights(cuda, 8, 640, 1408 // 2 + 8)
    w = fp8.Fp8Weight(q, s)
    starts = torch.tensor(np.cumsum([0] + counts), dtype=torch.int32, device=cuda)
    x = torch.randn(sum(counts), 640, device=cuda).bfloat16()
    g = torch.randn(sum(counts), q.shape[2], device=cuda).bfloat16()
    y = fp8.grouped_fp8_matmul(x, w, starts)
    b = fp8.grouped_fp8_matmul_backward(g, w, starts)
    xv, gv = value(*plain_rows(x)), value(*plain_rows(g))
    for e in range(8):
        a, z = int(starts[e]), int(starts[e + 1])
        wv = weight_value(q[e], s[e])
        check(y[a:z], xv[a:z], wv, 5)
        check(b[a:z], gv[a:z], wv.t(), 6)


# ------------------------------------------------------------------ how it is called
def test_streams_and_graphs(cuda):
    import torch
    from aethermoe_b200 import fp8
    q, s = weights(cuda, 4, 512, 640)
    w = fp8.Fp8Weight(q, s)
    starts = torch.tensor([0, 30, 31, 100, 170], dtype=torch.int32, device=cuda)
    x = torch.randn(170, 512, device=cuda).bfloat16()

    def step():
        h = fp8.grouped_fp8_matmul(x, w, starts, relu=True)
        return h, fp8.grouped_fp8_matmul_backward(h, w, starts), fp8.fp8_matmul(x[:3], w, 2), fp8.quantize_fp8(x).scale
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = fp8.grouped_fp8_matmul(x, w, starts, relu=True, stream=side)
    side.synchronize()
    assert torch.equal(got, want[0])
    leaf = x.clone().requires_grad_()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one = step()
        with pytest.raises(RuntimeError, match="captured"):
            fp8.fp8_matmul(leaf, w)
    with torch.cuda.graph(other):
        two = step()
    x.copy_(torch.randn(170, 512, device=cuda))
    want = step()
    graph.replay()
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.current_stream())
        other.replay()
    side.synchronize()
    torch.cuda.synchronize()
    for a, b, c in zip(one, two, want):
        assert torch.equal(a, c) and torch.equal(b, c)


def test_packing(cuda):
    """From the host and from strided device tensors, with the caller's device kept."""
    import torch
    from aethermoe_b200 import _lib, fp8
    q, s = weights(cuda, 2, 200, 130)
    x = torch.randn(20, 200, device=cuda)
    want = fp8.fp8_matmul(x, fp8.Fp8Weight(q, s), 1)
    assert torch.equal(fp8.fp8_matmul(x, fp8.Fp8Weight(q.cpu(), s.cpu()), 1), want)
    turned = q.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(torch.float8_e4m3fn)
    assert torch.equal(fp8.fp8_matmul(x, fp8.Fp8Weight(turned, s), 1), want)
    w = fp8.Fp8Weight(q[0], s[0])
    assert (w.G, w.K, w.N) == (1, 200, 130)
    w.close()
    with pytest.raises(ValueError, match="closed"):
        fp8.fp8_matmul(x, w)


def test_refusals_on_the_device(cuda):
    import torch
    from aethermoe_b200 import _lib, fp8
    q, s = weights(cuda, 2, 256, 128)
    w = fp8.Fp8Weight(q, s)
    x = torch.randn(8, 256, device=cuda)
    with pytest.raises(ValueError, match="columns"):
        fp8.fp8_matmul(x[:, :200], w)
    with pytest.raises(ValueError, match="group 2"):
        fp8.fp8_matmul(x, w, 2)
    with pytest.raises(ValueError, match="overlaps"):
        fp8.fp8_matmul(x, w, out=x[:, :128])
    with pytest.raises(ValueError, match="starts"):
        fp8.grouped_fp8_matmul(x, w, torch.zeros(4, dtype=torch.int32, device=cuda))
    with pytest.raises(ValueError, match="dtype"):
        fp8.fp8_matmul(x, w, out_dtype=torch.float16)
    with pytest.raises(RuntimeError, match="no gradient"):
        fp8.quantize_fp8(x.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="no gradient"):
        fp8.quantize_fp8_weight(x.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="autograd"):
        fp8.fp8_matmul(x.clone().requires_grad_(), w, out=torch.empty(8, 128, device=cuda))
    L = _lib.lib()
    out = torch.empty(8, 128, device=cuda)
    rows = fp8.quantize_fp8(x)

    def call(group=0, x=rows.q.data_ptr(), dt=_lib.E4M3, ldx=256, xs=rows.scale.data_ptr(), lds=4, M=8, out=out.data_ptr(),
             od=_lib.F32, ldo=128, ws=None, wb=0):
        return L.aem_fp8gemm(w.handle, group, 0, x, dt, ldx, xs, lds, M, out, od, ldo, ws, wb, None)
    for bad in (dict(group=-1), dict(group=2), dict(M=-1), dict(dt=5), dict(ldx=255), dict(ldx=240), dict(xs=None),
                dict(lds=1), dict(lds=3), dict(out=None), dict(x=None), dict(od=_lib.E4M3), dict(ldo=127),
                dict(x=rows.q.data_ptr() + 1), dict(dt=_lib.F32), dict(dt=_lib.F32, xs=None, ws=out.data_ptr(), wb=8)):
        assert call(**bad) == _lib.AEM_EINVAL, bad
    assert call(M=0) == _lib.AEM_OK and call() == _lib.AEM_OK
    torch.cuda.synchronize()
    assert torch.equal(out, fp8.fp8_matmul(x, w))
    assert fp8.fp8_matmul(x[:0], w).shape == (0, 128)


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("T", [1, 37, 900])
def test_a_layer_step(cuda, T):
    """Routing, dispatch, both expert products, combine, and the way back: every part
    against the plain form of what the part before it gave."""
    import torch
    from aethermoe_b200 import dispatch as D
    from aethermoe_b200 import fp8, routing
    from test_routing_gpu import check_route
    E, k, d, f = 16, 4, 256, 320
    up, down = weights(cuda, E, d, f, seed=1), weights(cuda, E, f, d, seed=2)
    U, V = fp8.Fp8Weight(*up), fp8.Fp8Weight(*down)
    x = torch.randn(T, d, device=cuda).requires_grad_()
    router = (torch.randn(d, E, device=cuda) / 16).requires_grad_()
    logits = x @ router
    how = dict(k=k, score="sigmoid", groups=4, top_groups=2, group_top=2, renormalize=True, scale=2.5)
    ids, w = routing.route_tokens(logits, **how)
    check_route(logits.detach(), ids, w.detach(), how)
    rows, order = D.dispatch(x, ids, E)
    a = fp8.grouped_fp8_matmul(rows, U, order.starts)
    h = torch.relu(a)
    y = fp8.grouped_fp8_matmul(h, V, order.starts)
    out = D.combine(y, w, order)
    kept = [logits, rows, a, h, y, w]
    for t in kept:
        t.retain_grad()
    g = torch.randn_like(out)
    out.backward(g)
    starts = order.starts.tolist()
    for e in range(E):
        i, j = starts[e], starts[e + 1]
        if i == j:
            continue
        uv, vv = weight_value(up[0][e], up[1][e]), weight_value(down[0][e], down[1][e])
        check(a.detach()[i:j], value(*plain_rows(rows.detach()[i:j])), uv, blocks(d))
        check(y.detach()[i:j], value(*plain_rows(h.detach()[i:j])), vv, blocks(f))
        check(h.grad[i:j], value(*plain_rows(y.grad[i:j])), vv.t(), blocks(d))
        check(rows.grad[i:j], value(*plain_rows(a.grad[i:j])), uv.t(), blocks(f))
    assert torch.equal(logits.grad, routing.route_tokens_backward(w.grad, logits.detach(), ids, score="sigmoid",
                                                                  renormalize=True, scale=2.5))
    assert torch.isfinite(x.grad).all() and torch.isfinite(router.grad).all() and router.grad.abs().max() > 0
