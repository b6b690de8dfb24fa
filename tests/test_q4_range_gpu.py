"""Rows of any range through the products with 4-bit weights: small elements
beside large ones lose nothing, on every row tile.

Tolerance: that of ``test_q4_gpu`` without its allowance for what is cut off,
and for elements that are added apart a chain of 32 fused multiply-adds, one
rounding for the scaled weight and one for each of the K / 32 parts and their
sum: (K / 32 + 34) * 2^-24 of the sum of magnitudes more.
"""
import pytest

from test_q4_gpu import HALF_BF16, weights

pytestmark = pytest.mark.gpu

ROWS = [1, 2, 3, 4, 5, 6, 8, 10, 11, 13, 16, 17, 21, 40, 70]


def check(got, x, q, s, gs):
    import torch
    K = x.shape[1]
    w = q.double() * s.double().repeat_interleave(gs, 0)[:K]
    ref, A = x.double() @ w, 1.25 * (x.double().abs() @ w.abs())
    tol = (132 * 2.0 ** -23 + (s.shape[0] + 15 + K / 32 + 34) * 2.0 ** -24) * A
    if got.dtype == torch.bfloat16:
        tol = tol + HALF_BF16 * (ref.abs() + tol)
    bad = ~((got.double() - ref).abs() <= tol)
    assert not bad.any(), ((got.double() - ref).abs()[bad][:4], tol[bad][:4], bad.nonzero()[:4])


@pytest.mark.parametrize("gs", [32, 64, 128])
@pytest.mark.parametrize("xdt", ["float32", "bfloat16"])
@pytest.mark.parametrize("K,N", [(192, 40), (3000, 300)])
@pytest.mark.parametrize("M", ROWS)
def test_every_bit_of_every_element_takes_part(cuda, M, K, N, xdt, gs):
    """One weight of 1 picks an element out, so the product must be that element,
    whatever else its row holds: 200 binary orders of magnitude, the largest
    float32, infinity's neighbours, zeros."""
    import torch
    from aethermoe_b200 import q4
    xdt = getattr(torch, xdt)
    g = torch.Generator(device=cuda).manual_seed(M * K + gs)
    q = torch.zeros(K, N, device=cuda, dtype=torch.int8)
    k = torch.randint(0, K, (N,), device=cuda, generator=g)
    q[k, torch.arange(N, device=cuda)] = 1
    w = q4.Q4Weight(q, torch.ones(-(-K // gs), N, device=cuda), gs)

    def same(x):
        x = x.to(xdt)
        assert torch.equal(q4.q4_matmul(x, w, out_dtype=torch.float32), x[:, k].float())
        starts = torch.tensor([0, M], dtype=torch.int32, device=cuda)
        assert torch.equal(q4.grouped_q4_matmul(x, w, starts, out_dtype=torch.float32), x[:, k].float())

    x = torch.randn(M, K, device=cuda, generator=g)
    same(x)
    same(x * torch.logspace(-36, 36, M, device=cuda)[:, None])  # each row its own size
    for span in (7, 8, 20, 24, 26, 30, 48, 200):  # around and past the windows' ends
        e = torch.randint(-span // 2, span - span // 2 + 1, (M, K), device=cuda, generator=g)
        same(torch.ldexp(x, e.float()))
    y = x * torch.logspace(-30, 30, K, device=cuda)
    y[0] = 3.3e38  # finite in both types
    y[M - 1, ::3] = 0
    same(y)


@pytest.mark.parametrize("order", [10, 20, 40, 90])
@pytest.mark.parametrize("xdt", ["float32", "bfloat16"])
@pytest.mark.parametrize("K,N,gs", [(4096, 520, 64), (640, 96, 32), (14336, 40, 128), (1999, 130, 128)])
def test_small_elements_beside_outlier_channels(cuda, K, N, gs, xdt, order):
    """Two channels 2^order larger than the rest; half of the columns have no weight
    there, so their sums hold small elements alone."""
    import torch
    from aethermoe_b200 import q4
    xdt = getattr(torch, xdt)
    q, s = weights(cuda, 1, K, N, gs, torch.float32, seed=K + order)
    q[:, 17, ::2] = q[:, K - 5, ::2] = 0
    w = q4.Q4Weight(q[0], s[0], gs)
    for M in (1, 2, 4, 5, 9, 16, 30, 64):
        x = torch.randn(M, K, device=cuda)
        x[:, 17] *= 2.0 ** order
        x[:, K - 5] *= 2.0 ** order
        x[M // 2] = torch.randn(K, device=cuda)  # an ordinary row among them
        x = x.to(xdt)
        check(q4.q4_matmul(x, w, out_dtype=torch.float32), x, q[0], s[0], gs)
        check(q4.q4_matmul(x, w, out_dtype=torch.bfloat16), x, q[0], s[0], gs)


@pytest.mark.parametrize("xdt", ["float32", "bfloat16"])
@pytest.mark.parametrize("sdt", ["float32", "bfloat16"])
@pytest.mark.parametrize("gs", [32, 128])
@pytest.mark.parametrize("most", [2, 7, 30])
def test_groups_with_outlier_rows(cuda, most, gs, sdt, xdt):
    """Ragged groups, rows of every range among them, infinities and NaN beside."""
    import torch
    from aethermoe_b200 import q4
    G, K, N = 24, 1100, 200
    q, s = weights(cuda, G, K, N, gs, getattr(torch, sdt), seed=most)
    w = q4.Q4Weight(q, s, gs)
    counts = torch.randint(0, most + 1, (G,), generator=torch.Generator().manual_seed(most + gs))
    starts = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)])
    M = int(starts[-1])
    e = torch.randint(0, 2, (M, K), device=cuda) * torch.randint(0, 70, (M, 1), device=cuda)
    x = torch.ldexp(torch.randn(M, K, device=cuda), e.float()).to(getattr(torch, xdt))
    x[0, 3], x[M - 1, 7] = float("inf"), float("nan")
    out = q4.grouped_q4_matmul(x, w, starts.int().to(cuda), out_dtype=torch.float32)
    for g in range(G):
        a, b = int(starts[g]), int(starts[g + 1])
        rows = [r for r in range(a, b) if 0 < r < M - 1]
        if rows:
            check(out[rows], x[rows], q[g], s[g].float(), gs)
    first = int((starts[1:] > 0).nonzero()[0])
    col = (q[first, 3] != 0)
    assert (out[0, col] == torch.sign(q[first, 3, col].float()) * float("inf")).all()
    assert out[0, ~col].isnan().all() and out[M - 1].isnan().all()  # infinity times a weight of zero, as in x @ w
    again = q4.grouped_q4_matmul(x, w, starts.int().to(cuda), out_dtype=torch.float32)
    assert torch.equal(again[1:M - 1], out[1:M - 1])


@pytest.mark.parametrize("xdt", ["float32", "bfloat16"])
@pytest.mark.parametrize("M", [1, 4, 12, 40])
def test_ranges_that_change_under_a_captured_call(cuda, M, xdt):
    """A graph captured on ordinary rows, replayed on rows of any range and back."""
    import torch
    from aethermoe_b200 import q4
    K, N = 2500, 260
    q, s = weights(cuda, 1, K, N, 64, torch.bfloat16, seed=M)
    w = q4.Q4Weight(q[0], s[0], 64)
    x = torch.randn(M, K, device=cuda).to(getattr(torch, xdt))
    q4.q4_matmul(x, w)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = q4.q4_matmul(x, w, out_dtype=torch.float32)
    for span in (0, 60, 0, 26):
        e = torch.randint(0, span + 1, (M, K), device=cuda).float()
        x.copy_(torch.ldexp(torch.randn(M, K, device=cuda), e))
        g.replay()
        check(out, x, q[0], s[0].float(), 64)
        assert torch.equal(out, q4.q4_matmul(x, w, out_dtype=torch.float32))
