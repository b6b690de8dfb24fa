"""4-bit quantisation and the products with 4-bit weights on the GPU, against a
plain implementation in 64 bits.

Tolerance of a product with A = sum_k |scale q x|: an MMA adds 32 products to
its accumulator, each aligned to the largest with at least 24 bits, so it
loses at most 33 * 2^-23 of the magnitudes it adds, and a scale group is at
most 4 MMAs: 132 * 2^-23 A.  The terms' sums (7), the groups' (ceil(K /
group) of them), the warpgroups' (1) and the cluster's (7) add up to
(groups + 15) * 2^-24 A, truncated terms' magnitudes add to at most 1.25 times
the value's.  What the terms cut off is under 2^-30 of the row's largest
magnitude for each k.  A bf16 result adds 2^-8 of its value.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HALF_BF16 = 2.0 ** -8


def weights(cuda, G, K, N, gs, sdt, seed=0, low=-7):
    import torch
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    q = torch.randint(low, 8, (G, K, N), device=cuda, dtype=torch.int8, generator=g)
    s = (torch.rand(G, -(-K // gs), N, device=cuda, generator=g) + 0.25).to(sdt)
    return q, s


def product(x, q, s, gs):
    """(sum, sum of magnitudes and what the terms may cut off, as a share of
    them, in units of the tolerance) in 64 bits."""
    w = q.double() * s.double().repeat_interleave(gs, 0)[:q.shape[0]]
    x = x.double()
    cut = 2.0 ** -30 * x.abs().amax(1, keepdim=True) * w.abs().sum(0)
    return x @ w, 1.25 * (x.abs() @ w.abs()) + cut / (132 * 2.0 ** -23)


def check(got, ref, A, KB):
    import torch
    tol = (132 * 2.0 ** -23 + (KB + 15) * 2.0 ** -24) * A
    if got.dtype == torch.bfloat16:
        tol = tol + HALF_BF16 * (ref.abs() + tol)
    bad = ~((got.double() - ref).abs() <= tol)
    assert not bad.any(), ((got.double() - ref).abs()[bad][:4], tol[bad][:4])


SIZES = [(1, 1, 1), (5, 7, 3), (64, 16, 1), (64, 32, 8), (100, 50, 9), (128, 33, 16), (333, 47, 17),
         (1000, 100, 33), (2048, 96, 64), (2056, 130, 65), (4096, 64, 2), (8200, 31, 7), (130, 1000, 131)]


@pytest.mark.parametrize("gs", [32, 64, 128])
@pytest.mark.parametrize("xdt,sdt", [("bfloat16", "bfloat16"), ("float32", "float32"),
                                     ("bfloat16", "float32"), ("float32", "bfloat16")])
@pytest.mark.parametrize("K,N,M", SIZES)
def test_product(cuda, K, N, M, gs, xdt, sdt):
    import torch
    from aethermoe_b200 import q4
    xdt, sdt = getattr(torch, xdt), getattr(torch, sdt)
    q, s = weights(cuda, 2, K, N, gs, sdt, seed=K + N)
    w = q4.Q4Weight(q, s, gs)
    x = torch.randn(M, K, device=cuda).to(xdt)
    for group in range(2):
        ref, A = product(x, q[group], s[group], gs)
        for odt in (torch.float32, torch.bfloat16):
            check(q4.q4_matmul(x, w, group, out_dtype=odt), ref, A, s.shape[1])


def test_float32_activations_take_part_in_full(cuda):
    """One weight of 1 picks x itself out: every bit of it within a factor of
    2^7 of the row's largest magnitude, and all but 2^-30 of that largest
    magnitude at any range."""
    import torch
    from aethermoe_b200 import q4
    K, N = 192, 40
    q = torch.zeros(K, N, device=cuda, dtype=torch.int8)
    k = torch.randint(0, K, (N,), device=cuda)
    q[k, torch.arange(N, device=cuda)] = 1
    w = q4.Q4Weight(q, torch.ones(K // 64, N, device=cuda), 64)
    x = (torch.rand(21, K, device=cuda) * 126 + 1.0001) * (torch.randint(0, 2, (21, K), device=cuda) * 2 - 1)
    x *= torch.logspace(-36, 36, 21, device=cuda)[:, None]  # each row its own size
    assert torch.equal(q4.q4_matmul(x, w), x[:, k])
    x = torch.randn(21, K, device=cuda) * torch.logspace(-30, 30, K, device=cuda)
    x[0, :] = 3.4028234e38  # the largest float32
    off = (q4.q4_matmul(x, w).double() - x[:, k].double()).abs()
    assert (off <= 2.0 ** -30 * x.double().abs().amax(1, keepdim=True)).all()
    # bf16: every bit within 2^23
    x = (torch.randn(40, K, device=cuda).bfloat16().float() * torch.exp2(torch.randint(0, 20, (40, K), device=cuda).float())).bfloat16()
    big = x.float().abs().amax(1, keepdim=True)
    x = torch.where(x.float().abs() * 2.0 ** 23 < big, torch.zeros_like(x), x)
    assert torch.equal(q4.q4_matmul(x, w), x[:, k])


def test_products_are_exact_on_whole_numbers(cuda):
    """Small whole numbers: every sum is exact, so results are equal bit for bit."""
    import torch
    from aethermoe_b200 import q4
    for K, N, gs in ((4096, 256, 128), (1472, 352, 32), (14336, 64, 64)):
        q = torch.randint(-7, 8, (K, N), device=cuda, dtype=torch.int8)
        s = torch.randint(1, 4, (-(-K // gs), N), device=cuda).float()
        w = q4.Q4Weight(q, s, gs)
        for M in (1, 8, 20, 64):
            x = torch.randint(-4, 5, (M, K), device=cuda).float()
            ref, _ = product(x, q, s, gs)
            assert torch.equal(q4.q4_matmul(x, w).double(), ref)
            assert torch.equal(q4.q4_matmul(x.bfloat16(), w, out_dtype=torch.float32).double(), ref)


@pytest.mark.parametrize("xdt", ["bfloat16", "float32"])
@pytest.mark.parametrize("G,K,N,gs,counts", [
    (1, 64, 32, 32, [3]),
    (4, 128, 48, 128, [0, 5, 0, 1]),
    (8, 256, 64, 64, [0] * 7 + [2]),
    (5, 200, 33, 32, [9, 0, 17, 64, 1]),
    (64, 320, 32, 64, [1] * 64),
    (256, 64, 16, 32, [i % 5 for i in range(256)]),
    (3, 192, 40, 64, [0, 200, 0]),
    (17, 128, 16, 128, [0] * 17),
])
def test_grouped_product(cuda, G, K, N, gs, counts, xdt):
    import torch
    from aethermoe_b200 import q4
    xdt = getattr(torch, xdt)
    q, s = weights(cuda, G, K, N, gs, torch.float32, seed=G)
    w = q4.Q4Weight(q, s, gs)
    extra = 6  # rows outside every group
    starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    M = int(starts[-1]) + extra
    x = torch.randn(M, K, device=cuda).to(xdt)
    x[int(starts[-1]):] = float("nan")
    st = torch.from_numpy(starts).to(cuda)
    for relu in (False, True):
        out = torch.full((M, N), 7.0, device=cuda, dtype=xdt)
        q4.grouped_q4_matmul(x, w, st, relu=relu, out=out)
        for g in range(G):
            a, b = starts[g], starts[g + 1]
            if a == b:
                continue
            ref, A = product(x[a:b], q[g], s[g], gs)
            check(out[a:b], ref.clamp(min=0) if relu else ref, A, s.shape[1])
        assert (out[int(starts[-1]):] == 7).all()


def test_groups_that_start_late_or_end_out_of_range(cuda):
    import torch
    from aethermoe_b200 import q4
    q, s = weights(cuda, 3, 64, 32, 64, torch.float32)
    w = q4.Q4Weight(q, s, 64)
    x = torch.randn(10, 64, device=cuda)
    out = torch.full((10, 32), 7.0, device=cuda)
    q4.grouped_q4_matmul(x, w, torch.tensor([2, 4, 6, 99], dtype=torch.int32, device=cuda), out=out)
    assert (out[:2] == 7).all()
    for g, (a, b) in enumerate(((2, 4), (4, 6), (6, 10))):
        ref, A = product(x[a:b], q[g], s[g], 64)
        check(out[a:b], ref, A, 1)
    out.fill_(7)
    q4.grouped_q4_matmul(x, w, torch.tensor([-5, -2, 3, 1], dtype=torch.int32, device=cuda), out=out)
    ref, A = product(x[:3], q[1], s[1], 64)
    check(out[:3], ref, A, 1)
    assert (out[3:] == 7).all()


@pytest.mark.parametrize("xdt", ["bfloat16", "float32"])
def test_strides_and_alignment(cuda, xdt):
    import torch
    from aethermoe_b200 import q4
    xdt = getattr(torch, xdt)
    for K, N, off, pad in ((128, 48, 8, 8), (128, 48, 1, 3), (136, 31, 4, 0), (64, 32, 0, 1)):
        q, s = weights(cuda, 1, K, N, 32, torch.float32)
        w = q4.Q4Weight(q[0], s[0], 32)
        big = torch.randn(11, off + K + pad, device=cuda).to(xdt)
        x = big[:, off:off + K]
        ref, A = product(x, q[0], s[0], 32)
        buf = torch.full((11, off + N + pad), 7.0, device=cuda)
        q4.q4_matmul(x, w, out=buf[:, off:off + N])
        check(buf[:, off:off + N], ref, A, s.shape[1])
        assert (buf[:, :off] == 7).all() and (buf[:, off + N:] == 7).all()
        xt = torch.randn(K, 11, device=cuda).to(xdt).t()
        ref, A = product(xt, q[0], s[0], 32)
        check(q4.q4_matmul(xt, w, out_dtype=torch.float32), ref, A, s.shape[1])
        one = torch.randn(1, K, device=cuda).to(xdt).expand(5, K)
        ref, A = product(one, q[0], s[0], 32)
        check(q4.q4_matmul(one, w, out_dtype=torch.float32), ref, A, s.shape[1])


@pytest.mark.parametrize("xdt", ["bfloat16", "float32"])
def test_infinities_and_nan_stay_in_their_rows(cuda, xdt):
    import torch
    from aethermoe_b200 import q4
    xdt = getattr(torch, xdt)
    K, N = 256, 64
    q, s = weights(cuda, 1, K, N, 64, torch.float32, low=1)  # no zero weight: inf stays inf
    w = q4.Q4Weight(q[0], s[0], 64)
    x = torch.randn(12, K, device=cuda).to(xdt)
    x[3, 5], x[4, 77], x[5, 200] = float("inf"), float("nan"), -float("inf")
    out = q4.q4_matmul(x, w, out_dtype=torch.float32)
    assert (out[3] == float("inf")).all() and out[4].isnan().all() and (out[5] == -float("inf")).all()
    rest = [i for i in range(12) if i not in (3, 4, 5)]
    ref, A = product(x[rest], q[0], s[0], 64)
    check(out[rest], ref, A, 4)
    relu = q4.grouped_q4_matmul(x, w, torch.tensor([0, 12], dtype=torch.int32, device=cuda), relu=True)
    assert (relu[3] == float("inf")).all() and relu[4].isnan().all() and (relu[5] == 0).all()


@pytest.mark.parametrize("wdt,sdt", [("float32", "float32"), ("float32", "bfloat16"),
                                     ("bfloat16", "float32"), ("bfloat16", "bfloat16")])
@pytest.mark.parametrize("shape", [(1, 1), (31, 5), (32, 128), (129, 130), (1000, 36), (3, 70, 12), (2, 256, 64)])
@pytest.mark.parametrize("gs", [32, 64, 128])
def test_quantize(cuda, shape, gs, wdt, sdt):
    import torch
    from aethermoe_b200 import q4
    wdt, sdt = getattr(torch, wdt), getattr(torch, sdt)
    g = torch.Generator().manual_seed(sum(shape))
    w = torch.randn(*shape, generator=g) * 0.02
    w[..., : shape[-2] // 2, 0] = 0.0  # a column that is zero in its first groups
    w = w.to(wdt)
    q, s = q4.quantize_q4(w.to(cuda), gs, sdt)
    K = shape[-2]
    kb = -(-K // gs)
    f = w.float().reshape(-1, K, shape[-1])
    pad = torch.nn.functional.pad(f.abs(), (0, 0, 0, kb * gs - K)).reshape(f.shape[0], kb, gs, -1)
    want = (pad.amax(2) / 7.0).clamp(min=1e-12).to(sdt)  # CPU: IEEE division
    wq = torch.round(f / want.float().repeat_interleave(gs, 1)[:, :K]).clamp(-7, 7).to(torch.int8)
    assert s.dtype == sdt and torch.equal(s.cpu().reshape(want.shape), want)
    assert torch.equal(q.cpu().reshape(wq.shape), wq)


def test_quantized_product_is_near_the_unquantized(cuda):
    """Half a quantisation step per weight: |w - q s| <= s / 2 (and the clipped
    7.0x of a scale that bf16 rounded down: 2^-8 of 7 steps)."""
    import torch
    from aethermoe_b200 import q4
    w = torch.randn(512, 96, device=cuda) * 0.02
    for sdt, half in ((torch.float32, 0.5), (torch.bfloat16, 0.5)):
        q, s = q4.quantize_q4(w, 64, sdt)
        full = s.double().repeat_interleave(64, 0)
        assert ((w.double() - q.double() * full).abs() <= half * full * (1 + 1e-6)).all()
        weight = q4.Q4Weight(q, s, 64)
        x = torch.randn(6, 512, device=cuda)
        ref, A = product(x, q, s, 64)
        check(q4.q4_matmul(x, weight), ref, A, 8)


def test_host_and_device_packs_agree(cuda):
    import torch
    from aethermoe_b200 import _lib, q4
    q, s = weights(cuda, 3, 100, 37, 32, torch.bfloat16)
    a, b = q4.Q4Weight(q, s, 32), q4.Q4Weight(q.cpu(), s.cpu(), 32)
    c = q4.Q4Weight(q.cpu().numpy(), s.float().cpu().numpy(), 32)
    x = torch.randn(4, 100, device=cuda)
    for g in range(3):
        assert torch.equal(q4.q4_matmul(x, a, g), q4.q4_matmul(x, b, g))
        assert torch.equal(q4.q4_matmul(x, a, g), q4.q4_matmul(x, c, g))
    bad = q.clone()
    bad[1, 50, 20] = -8
    with pytest.raises(ValueError, match="-7, 7"):
        q4.Q4Weight(bad, s, 32)
    assert _lib.lib().aem_device_status(None) == _lib.AEM_OK


def test_refusals(cuda):
    import torch
    from aethermoe_b200 import q4
    q, s = weights(cuda, 2, 64, 32, 32, torch.float32)
    w = q4.Q4Weight(q, s, 32)
    x = torch.zeros(2, 64, device=cuda)
    for bad in (lambda: q4.q4_matmul(x[:, :63], w), lambda: q4.q4_matmul(x, w, 2), lambda: q4.q4_matmul(x, w, -1),
                lambda: q4.q4_matmul(x.half(), w), lambda: q4.q4_matmul(x.cpu(), w),
                lambda: q4.q4_matmul(x, w, out=torch.zeros(2, 31, device=cuda)),
                lambda: q4.q4_matmul(x, w, out=torch.zeros(1, 32, device=cuda).expand(2, 32)),
                lambda: q4.grouped_q4_matmul(x, w, torch.zeros(2, dtype=torch.int32, device=cuda)),
                lambda: q4.grouped_q4_matmul(x, w, torch.zeros(3, device=cuda))):
        with pytest.raises(ValueError):
            bad()
    assert q4.q4_matmul(x[:0], w).shape == (0, 32)
    w.close()
    with pytest.raises(ValueError, match="closed"):
        q4.q4_matmul(x, w)


def test_captured_other_stream_and_repeats(cuda):
    import torch
    from aethermoe_b200 import q4
    q, s = weights(cuda, 4, 2048, 96, 64, torch.bfloat16)
    w = q4.Q4Weight(q, s, 64)
    starts = torch.tensor([0, 3, 3, 20, 30], dtype=torch.int32, device=cuda)
    x = torch.randn(30, 2048, device=cuda).bfloat16()
    one, many = q4.q4_matmul(x, w, 1), q4.grouped_q4_matmul(x, w, starts)
    side = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for st in side:
        st.wait_stream(torch.cuda.current_stream())
        got.append((q4.q4_matmul(x, w, 1, stream=st), q4.grouped_q4_matmul(x, w, starts, stream=st)))
    torch.cuda.synchronize()
    for a, b in got:
        assert torch.equal(a, one) and torch.equal(b, many)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a = q4.q4_matmul(x, w, 1)
        b = q4.grouped_q4_matmul(x, w, starts)
    for _ in range(3):
        x.normal_()
        starts[1:4] = torch.sort(torch.randint(0, 31, (3,), device=cuda)).values.int()
        g.replay()
        assert torch.equal(a, q4.q4_matmul(x, w, 1)) and torch.equal(b, q4.grouped_q4_matmul(x, w, starts))


def test_weights_past_32_bit_offsets(cuda):
    import torch
    from aethermoe_b200 import q4
    G, K, N = 256, 4096, 4608  # 4.8e9 weights
    q = torch.empty(G, K, N, device=cuda, dtype=torch.int8)
    for g in range(0, G, 32):
        q[g:g + 32].random_(-7, 8)
    s = torch.rand(G, K // 128, N, device=cuda) + 0.5
    w = q4.Q4Weight(q, s, 128)
    x = torch.randn(3, K, device=cuda)
    for g in (0, 130, 255):
        ref, A = product(x, q[g], s[g], 128)
        check(q4.q4_matmul(x, w, g), ref, A, 32)
    starts = torch.zeros(G + 1, dtype=torch.int32, device=cuda)
    starts[G] = 3
    ref, A = product(x, q[255], s[255], 128)
    check(q4.grouped_q4_matmul(x, w, starts), ref, A, 32)


@pytest.mark.parametrize("T,k,E,d,f,dtype", [(1, 2, 8, 256, 384, "bfloat16"), (37, 3, 16, 192, 320, "float32"),
                                             (64, 6, 64, 128, 96, "bfloat16")])
def test_whole_expert_step(cuda, T, k, E, d, f, dtype):
    """Gating, dispatch, both expert products, combine: as a decoding step runs them.
    The order must be the gating's; the 64-bit step rounds where the kernels'
    outputs do, so each product is checked on the very rows that entered it."""
    import torch
    import aem_oracle as O
    from aethermoe_b200 import _lib, q4
    from aethermoe_b200 import dispatch as D
    dt = getattr(torch, dtype)
    rng = np.random.default_rng(T)
    gw = (rng.normal(size=(d, E)) / np.sqrt(d)).astype(np.float32)
    gate = _lib.Gate(gw, O.zipf_bias(E))
    x = torch.from_numpy(rng.normal(size=(T, d)).astype(np.float32)).to(cuda).to(dt)
    idx = torch.empty(T, k + 1, dtype=torch.int32, device=cuda)
    val = torch.empty(T, k, dtype=torch.float32, device=cuda)
    _lib.check(_lib.lib().aem_gating(gate.handle, x.data_ptr(), _lib.BF16 if dt == torch.bfloat16 else _lib.F32,
                                     T, k, 1, _lib.GATING_EXACT, idx.data_ptr(), val.data_ptr(),
                                     torch.cuda.current_stream().cuda_stream))
    oidx, oval = O.fused_gating(x.float().cpu().numpy(), gw, O.zipf_bias(E), k)
    np.testing.assert_array_equal(idx[:, :k].cpu().numpy(), oidx)
    qu, su = q4.quantize_q4(torch.randn(E, d, f, device=cuda) / d ** 0.5, 64)
    qd, sd = q4.quantize_q4(torch.randn(E, f, d, device=cuda) / f ** 0.5, 32, torch.bfloat16)
    up, down = q4.Q4Weight(qu, su, 64), q4.Q4Weight(qd, sd, 32)

    rows, order = D.dispatch(x, idx[:, :k], E)
    h = q4.grouped_q4_matmul(rows, up, order.starts, relu=True)
    y = q4.grouped_q4_matmul(h, down, order.starts, out_dtype=torch.float32)
    out = D.combine(y, val, order, out_dtype=dt)

    want = torch.zeros(T, d, dtype=torch.float64, device=cuda)
    size = torch.zeros_like(want)
    for t in range(T):
        for j in range(k):
            e, r = int(idx[t, j]), int(order.row_of[t, j])
            assert torch.equal(rows[r], x[t])
            hr, hA = product(x[t:t + 1], qu[e], su[e], 64)
            check(h[r:r + 1], hr.clamp(min=0), hA, su.shape[1])
            yr, yA = product(h[r:r + 1], qd[e], sd[e], 32)
            check(y[r:r + 1], yr, yA, sd.shape[1])
            want[t] += val[t, j].double() * y[r].double()
            size[t] += (val[t, j].double() * y[r].double()).abs()
    tol = k * 2.0 ** -24 * size
    if dt == torch.bfloat16:
        tol = tol + HALF_BF16 * (want.abs() + tol)
    assert ((out.double() - want).abs() <= tol).all()
