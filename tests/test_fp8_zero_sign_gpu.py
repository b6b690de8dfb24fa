"""8-bit quantisation on the GPU, byte for byte: the sign of a zero is that of the
quotient x / scale, for scales where it is computed in steps and where the
division itself is made."""
import pytest

from test_fp8_gpu import blocks, plain_rows

pytestmark = pytest.mark.gpu

TOPS = (448.0, 1.0, 3.1e-3, 1.3e-20, 1e-30, 2.0 ** -81, 1e-40, 5e20, 3e38)


def with_zeros(cuda, M, K, dt, seed=0):
    """Rows of zeros of both signs, of values that round to zero, of others, and one
    magnitude that sets the block's scale."""
    import torch
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    x = torch.randn(M, K, device=cuda, generator=g)
    kind = torch.randint(0, 4, (M, K), device=cuda, generator=g)
    x = torch.where(kind == 0, 0.0, torch.where(kind == 1, -0.0, torch.where(kind == 2, 1e-6 * x, x)))
    x = x / x.abs().amax(1, keepdim=True).clamp(min=2.0 ** -100)
    return (x * torch.tensor(TOPS, device=cuda).repeat(-(-M // len(TOPS)))[:M, None]).to(dt)


@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
@pytest.mark.parametrize("M,K", [(9, 128), (27, 300), (18, 2048), (45, 1)])
def test_bytes_of_rows(cuda, M, K, dt):
    import torch
    from aethermoe_b200 import fp8
    x = with_zeros(cuda, M, K, getattr(torch, dt), seed=K)
    if K > 1:
        assert (torch.signbit(x) & (x == 0)).any()
    rows = fp8.quantize_fp8(x)
    q, s = plain_rows(x)
    assert torch.equal(rows.scale, s)
    assert torch.equal(rows.q.view(torch.uint8), q.view(torch.uint8))


@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
@pytest.mark.parametrize("K,N", [(128, 128), (129, 257), (300, 132), (512, 1408)])
def test_bytes_of_weights(cuda, K, N, dt):
    import torch
    from aethermoe_b200 import fp8
    w = with_zeros(cuda, K, N, torch.float32, seed=N)
    w = (w / w.abs().amax(1, keepdim=True)).to(getattr(torch, dt))
    q, s = fp8.quantize_fp8_weight(w)
    p = torch.nn.functional.pad(w.float(), (0, -N % 128, 0, -K % 128)).reshape(blocks(K), 128, blocks(N), 128)
    want = p.abs().amax((1, 3))
    want = (want / torch.full_like(want, 448.0)).clamp(min=2.0 ** -126)
    pq = (p / want[:, None, :, None]).to(torch.float8_e4m3fn).reshape(blocks(K) * 128, -1)[:K, :N]
    assert torch.equal(s, want)
    assert torch.equal(q.view(torch.uint8), pq.contiguous().view(torch.uint8))


def test_a_row_of_negative_zeros(cuda):
    import torch
    from aethermoe_b200 import fp8
    rows = fp8.quantize_fp8(torch.full((2, 200), -0.0, device=cuda))
    assert (rows.q.view(torch.uint8) == 0x80).all()
    assert (rows.scale == 2.0 ** -126).all()
