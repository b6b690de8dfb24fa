"""The 8-bit products and the routing from logits where sizes change kernels or
pass 32 bits, on two streams at once, and rows that belong to no group.  Tolerances
as in ``test_fp8_gpu.py``."""
import numpy as np
import pytest

from test_fp8_gpu import blocks, check, plain_rows, value, weight_value, weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("K,N,M", [(4200, 4096, 2600), (5000, 4096, 600), (4096, 96, 300), (14336, 130, 100),
                                   (128, 14336, 700), (96, 520, 20000)])
def test_long_sums_and_many_tiles(cuda, K, N, M):
    """More than 32 blocks of the sum, odd numbers of them, several tiles for a pair of
    SMs, sums split over a cluster."""
    import torch
    from aethermoe_b200 import _lib, fp8
    q, s = weights(cuda, 1, K, N, seed=K)
    w = fp8.Fp8Weight(q[0], s[0])
    wv = weight_value(q[0], s[0])
    x, g = torch.randn(M, K, device=cuda).bfloat16(), torch.randn(M, N, device=cuda)
    check(fp8.fp8_matmul(x, w), value(*plain_rows(x)), wv, blocks(K))
    check(fp8.fp8_matmul_backward(g, w), value(*plain_rows(g)), wv.t(), blocks(N))
    _lib.check(_lib.lib().aem_device_status(None))


@pytest.mark.parametrize("K,N,counts", [(4096, 96, [100, 0, 130, 90]), (96, 4096, [70, 90, 1, 0]),
                                        (2048, 1408, [600, 0, 257, 255, 1, 900, 31, 33])])
def test_groups_of_either_kernel(cuda, K, N, counts):
    import torch
    from aethermoe_b200 import fp8
    G = len(counts)
    q, s = weights(cuda, G, K, N, seed=N)
    w = fp8.Fp8Weight(q, s)
    starts = torch.tensor(np.cumsum([2] + counts), dtype=torch.int32, device=cuda)
    M = int(starts[-1]) + 5
    x, g = torch.randn(M, K, device=cuda).bfloat16(), torch.randn(M, N, device=cuda).bfloat16()
    xv, gv = value(*plain_rows(x)), value(*plain_rows(g))
    for odt in (torch.bfloat16, torch.float32):
        y = torch.full((M, N), 9.0, device=cuda, dtype=odt)
        fp8.grouped_fp8_matmul(x, w, starts, out=y)
        b = torch.full((M, K), 9.0, device=cuda, dtype=odt)
        fp8.grouped_fp8_matmul_backward(g, w, starts, out=b)
        for e in range(G):
            i, j = int(starts[e]), int(starts[e + 1])
            if i < j:
                check(y[i:j], xv[i:j], weight_value(q[e], s[e]), blocks(K))
                check(b[i:j], gv[i:j], weight_value(q[e], s[e]).t(), blocks(N))
        assert (y[:2] == 9).all() and (y[M - 5:] == 9).all() and (b[:2] == 0).all() and (b[M - 5:] == 0).all()


def test_offsets_outside_the_rows_are_clamped(cuda):
    import torch
    from aethermoe_b200 import _lib, fp8
    q, s = weights(cuda, 3, 128, 128)
    w = fp8.Fp8Weight(q, s)
    for M in (40, 900):
        x = torch.randn(M, 128, device=cuda)
        good = torch.tensor([0, 7, 20, M], dtype=torch.int32, device=cuda)
        wild = torch.tensor([-5, 7, 20, M + 1000], dtype=torch.int32, device=cuda)
        assert torch.equal(fp8.grouped_fp8_matmul(x, w, wild), fp8.grouped_fp8_matmul(x, w, good))
        none = torch.full((4,), M + 9, dtype=torch.int32, device=cuda)
        out = torch.full((M, 128), 3.0, device=cuda)
        assert (fp8.grouped_fp8_matmul(x, w, none, out=out) == 3).all()
        assert (fp8.grouped_fp8_matmul_backward(x, w, none) == 0).all()
    _lib.check(_lib.lib().aem_device_status(None))


def test_two_streams_at_once(cuda):
    """Both kernels on two streams, weights shared: results as alone."""
    import torch
    from aethermoe_b200 import _lib, fp8
    q, s = weights(cuda, 1, 1024, 2048)
    w = fp8.Fp8Weight(q[0], s[0])
    xs = [torch.randn(M, 1024, device=cuda).bfloat16() for M in (5, 40, 100, 700, 1500)]
    want = [fp8.fp8_matmul(x, w) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for r in range(6):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] += [fp8.fp8_matmul(x, w) for x in (xs if i else xs[::-1])]
    torch.cuda.synchronize()
    for r in range(6):
        for k in range(5):
            assert torch.equal(got[1][5 * r + k], want[k]) and torch.equal(got[0][5 * r + k], want[4 - k])
    _lib.check(_lib.lib().aem_device_status(None))


def test_more_rows_than_a_grid_holds(cuda):
    import torch
    from aethermoe_b200 import fp8
    q, s = weights(cuda, 1, 16, 8)
    w = fp8.Fp8Weight(q[0], s[0])
    M = 65535 * 64 + 77
    x = torch.randn(M, 16, device=cuda).bfloat16()
    y = fp8.fp8_matmul(x, w)
    at = torch.cat([torch.arange(300), torch.arange(M - 300, M)]).to(cuda)
    check(y[at], value(*plain_rows(x[at])), weight_value(q[0], s[0]), 1)
    assert torch.isfinite(y).all()


def test_elements_past_32_bits(cuda):
    """More than 2^31 elements of x, of its quantised form, of out, and of the logits."""
    import torch
    from aethermoe_b200 import fp8, routing
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of free memory")
    M, K = (1 << 20) + 100, 2056
    x = torch.empty(M, K, device=cuda, dtype=torch.bfloat16).normal_()
    rows = fp8.quantize_fp8(x)
    at = torch.cat([torch.arange(50), torch.arange(M - 50, M)]).to(cuda)
    qq, ss = plain_rows(x[at])
    assert torch.equal(rows.scale[at], ss) and torch.equal(rows.q.view(torch.uint8)[at].view(torch.float8_e4m3fn).float(), qq.float())
    q, s = weights(cuda, 1, K, 16)
    w = fp8.Fp8Weight(q[0], s[0])
    y = fp8.fp8_matmul(rows, w)
    check(y[at], value(qq, ss), weight_value(q[0], s[0]), blocks(K))
    b = fp8.fp8_matmul_backward(y.bfloat16(), w)  # out of M x K elements
    check(b[at], value(*plain_rows(y[at].bfloat16())), weight_value(q[0], s[0]).t(), 1)
    del rows, y, b, x
    T, E = (1 << 23) + 5, 256
    x = torch.zeros(T, E, device=cuda, dtype=torch.bfloat16)
    x[:, 7] = 1.0
    x[-1, 200] = 2.0
    ids, wt = routing.route_tokens(x, 2, score="sigmoid")
    assert (ids[:-1, 0] == 7).all() and (ids[:-1, 1] == 0).all() and ids[-1].tolist() == [200, 7]
    g = routing.route_tokens_backward(torch.ones_like(wt), x, ids, score="sigmoid")
    assert (g[-1] != 0).sum() == 2 and (g[-2] != 0).sum() == 2 and float(g[-1, 200]) > 0


def test_rows_that_require_a_gradient_as_scales_are_refused(cuda):
    import torch
    from aethermoe_b200 import fp8
    rows = fp8.quantize_fp8(torch.randn(4, 128, device=cuda))
    with pytest.raises(RuntimeError, match="no gradient"):
        fp8.Fp8Rows(rows.q, rows.scale.clone().requires_grad_())
    q, s = weights(cuda, 1, 128, 128)
    with pytest.raises(RuntimeError, match="no gradient"):
        fp8.Fp8Weight(q, s.clone().requires_grad_())


def test_weights_packed_on_one_stream_are_used_on_another(cuda):
    import torch
    from aethermoe_b200 import fp8
    q, s = weights(cuda, 1, 2048, 4096)
    x = torch.randn(3, 2048, device=cuda)
    want = fp8.fp8_matmul(x, fp8.Fp8Weight(q, s))
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        w = fp8.Fp8Weight(q, s, stream=a)
        got = fp8.fp8_matmul(x, w, stream=b)
        b.synchronize()
        assert torch.equal(got, want)


@pytest.mark.parametrize("odt", ["bfloat16", "float32"])
@pytest.mark.parametrize("N", [520, 130, 47, 256])
def test_many_rows_into_rows_of_any_stride(cuda, N, odt):
    """20000 rows: the kernel for many rows, whose results leave by whole rows of 16-byte
    pieces where they can.  The same bits wherever they go, and nothing beside them."""
    import torch
    from aethermoe_b200 import _lib, fp8
    K, M, odt = 96, 20000, getattr(torch, odt)
    q, s = weights(cuda, 2, K, N, seed=N)
    w = fp8.Fp8Weight(q, s)
    x = torch.randn(M, K, device=cuda).bfloat16()
    starts = torch.tensor([0, 9001, M - 300], dtype=torch.int32, device=cuda)
    want, grouped = fp8.fp8_matmul(x, w, 1, out_dtype=odt), torch.full((M, N), 7.0, device=cuda, dtype=odt)
    check(want, value(*plain_rows(x)), weight_value(q[1], s[1]), blocks(K))
    fp8.grouped_fp8_matmul(x, w, starts, out=grouped)
    assert torch.equal(grouped[9001:M - 300], want[9001:M - 300]) and (grouped[M - 300:] == 7).all()
    for before, after in ((0, 8), (8, 0), (4, 4), (2, 2), (1, 0), (0, 3)):
        out = torch.full((M + 2, before + N + after), 7.0, device=cuda, dtype=odt)
        inner = out[1:M + 1, before:before + N]
        assert torch.equal(fp8.fp8_matmul(x, w, 1, out=inner), want), (before, after)
        fp8.grouped_fp8_matmul(x, w, starts, out=inner.fill_(7.0))
        assert torch.equal(inner, grouped), (before, after)
        inner.fill_(7.0)
        assert (out == 7).all(), (before, after)
    _lib.check(_lib.lib().aem_device_status(None))


@pytest.mark.parametrize("odt,N", [("bfloat16", 8192), ("float32", 8136)])
def test_more_tiles_than_are_looked_up_at_once(cuda, odt, N):
    """Some 260 tiles for a pair of SMs.  A row's results depend on no other row, so rows
    that repeat give the same bits wherever they lie."""
    import torch
    from aethermoe_b200 import _lib, fp8
    K, times = 64, 310
    q, s = weights(cuda, 2, K, N, seed=5)
    w = fp8.Fp8Weight(q, s)
    x = torch.randn(512, K, device=cuda)
    starts = torch.tensor([0, 512 * 7, 512 * times], dtype=torch.int32, device=cuda)
    y = fp8.grouped_fp8_matmul(x.repeat(times, 1), w, starts, out_dtype=getattr(torch, odt))
    xv = value(*plain_rows(x))
    for first, e in ((0, 0), (7, 1)):
        check(y[512 * first:512 * (first + 1)], xv, weight_value(q[e], s[e]), blocks(K))
    y = y.view(times, 512, N)
    for i in range(times):
        assert torch.equal(y[i], y[0 if i < 7 else 7]), i
    _lib.check(_lib.lib().aem_device_status(None))


@pytest.mark.parametrize("E,k,groups,top", [(256, 8, 8, 4), (64, 6, 4, 2), (60, 6, 4, 2), (16, 4, 2, 1)])
def test_route_with_many_near_ties(cuda, E, k, groups, top):
    """Every row needs the 64-bit choice: biases that undo the scores of one row's
    logits to a float32 rounding, for rows that differ from it in a few places."""
    import torch
    from aethermoe_b200 import routing
    from test_routing_gpu import check_route, plain_scores
    rng = np.random.default_rng(E)
    row = rng.normal(size=E).astype(np.float32)
    x = np.tile(row, (150, 1))
    for t in range(150):
        x[t, rng.integers(0, E, 3)] += rng.normal(size=3).astype(np.float32) * 1e-6
    x = torch.from_numpy(x).to(cuda)
    for score in ("softmax", "sigmoid"):
        bias = torch.from_numpy((1.0 - plain_scores(row[None].astype(np.float64), score)[0]).astype(np.float32)).to(cuda)
        for gt in (1, 2):
            how = dict(k=k, score=score, groups=groups, top_groups=top, group_top=gt, renormalize=True)
            ids, w = routing.route_tokens(x, bias=bias, **how)
            check_route(x, ids, w, dict(how, bias=bias.cpu().numpy()))
