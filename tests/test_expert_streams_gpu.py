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


@pytest.mark.parametrize("T,k,E,d", [(7, 2, 4, 16), (900, 3, 16, 72)])
def test_gradients_on_another_stream(cuda, monkeypatch, T, k, E, d):
    """Forward and backward of a step on ``stream``, called with another stream current:
    the backward kernels run there too, and their inputs are not reused meanwhile."""
    import torch
    from aethermoe_b200 import dispatch as D
    g = torch.Generator(device=cuda).manual_seed(T)
    ids = torch.randint(-1, E, (T, k), device=cuda, dtype=torch.int32, generator=g)
    x0 = torch.randn(T, d, device=cuda, generator=g)
    w0 = torch.rand(T, k, device=cuda, generator=g)
    go = torch.randn(T, d, device=cuda, generator=g)

    def step(stream):
        x, w = x0.clone().requires_grad_(), w0.clone().requires_grad_()
        if stream is not None:
            stream.wait_stream(torch.cuda.current_stream())
        rows, order = D.dispatch(x, ids, E, stream=stream)
        again = D.dispatch_rows(x, order, stream=stream)
        a, b = (D.combine(r, w, order, stream=stream) for r in (rows, again))
        if stream is not None:
            torch.cuda.current_stream().wait_stream(stream)
        del rows, order, again
        torch.autograd.backward([a, b], [go, 2 * go])
        del a, b
        return x.grad, w.grad
    want = step(None)
    side = torch.cuda.Stream()
    at = []
    handle = D._stream_handle
    monkeypatch.setattr(D, "_stream_handle", lambda dev: at.append(handle(dev)) or at[-1])
    for _ in range(5):
        keep = busy(cuda, 8)
        at.clear()
        got = step(side)
        with torch.cuda.stream(side):
            noise = [torch.full((n,), -1, device=cuda, dtype=torch.int32) for n in (2 * T * k + E + 1, T * k * d)]
        assert len(at) == 4 and set(at) == {side.cuda_stream}  # two calls of either backward pass
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        del keep, noise
