"""The expert operators on a stream that is not the current one: copies that a
call makes, gradients, and memory that the current stream reuses meanwhile."""
import pytest

pytestmark = pytest.mark.gpu


def busy(device, n=24):
    """Some milliseconds of work on the current stream."""
    import torch
    a = torch.randn(4096, 4096, device=device)
    for _ in range(n):
        a = a @ a * 1e-2
    return a


@pytest.mark.parametrize("wdt", ["float32", "bfloat16"])
@pytest.mark.parametrize("groups", [0, 3])
def test_strided_weights_on_another_stream(cuda, groups, wdt):
    """A transposed weight is copied, quantised and packed on ``stream`` in order,
    whatever the current stream is busy with and allocates afterwards."""
    import torch
    from aethermoe_b200 import q4
    g = torch.Generator(device=cuda).manual_seed(groups)
    shape = (groups, 1536, 2048) if groups else (1536, 2048)
    wt = (torch.randn(*shape, device=cuda, generator=g) * 0.02).to(getattr(torch, wdt))
    w = wt.transpose(-1, -2)
    want_q, want_s = q4.quantize_q4(w.contiguous(), 64)
    x = torch.randn(3, 2048, device=cuda, generator=g)
    want = q4.q4_matmul(x, q4.Q4Weight(want_q, want_s, 64))
    qt, st = want_q.transpose(-1, -2).contiguous(), want_s.transpose(-1, -2).contiguous()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(4):
        side.wait_stream(torch.cuda.current_stream())
        keep = busy(cuda)
        q, s = q4.quantize_q4(w, 64, stream=side)
        noise = [torch.full(shape, 7.0, device=cuda).to(w.dtype) for _ in range(3)]
        packed = q4.Q4Weight(qt.transpose(-1, -2), st.transpose(-1, -2), 64, stream=side)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(q, want_q) and torch.equal(s, want_s)
        assert torch.equal(q4.q4_matmul(x, packed), want)
        del keep, noise
