"""Argument checks of the dispatch, combine and 4-bit weight calls: refused
before any GPU work, so they run on any host."""
import ctypes

import numpy as np
import pytest
import torch

from aethermoe_b200 import _lib
from aethermoe_b200 import dispatch as D
from aethermoe_b200 import q4

P = 4096  # a pointer that no refused call follows
EINVAL = _lib.AEM_EINVAL


def L():
    return _lib.lib()


def test_dispatch_refusals():
    def call(x=P, dt=_lib.F32, ldx=8, d=8, ids=P, T=4, k=2, st=2, sk=1, E=8, rows=P, ldr=8, starts=P,
             row_of=P, unit_of=P, ws=None, wb=0):
        return L().aem_dispatch(x, dt, ldx, d, ids, T, k, st, sk, E, rows, ldr, starts, row_of, unit_of,
                                ws, wb, None)
    for bad in (dict(x=None), dict(rows=None), dict(ids=None), dict(starts=None), dict(row_of=None),
                dict(unit_of=None), dict(T=-1), dict(k=0), dict(k=65), dict(E=0), dict(E=257),
                dict(dt=7), dict(d=0), dict(ldr=7), dict(ldx=-1), dict(st=-1), dict(sk=-1),
                dict(T=1 << 30, k=2), dict(T=2000, ws=P, wb=8)):
        assert call(**bad) == EINVAL, bad
    assert L().aem_token_sort(None, 4, 2, 2, 1, 8, P, P, P, None, 0, None) == EINVAL


def test_dispatch_rows_refusals():
    def call(x=P, dt=_lib.F32, ldx=8, d=8, row_of=P, starts=P, T=4, k=2, E=8, rows=P, ldr=8):
        return L().aem_dispatch_rows(x, dt, ldx, d, row_of, starts, T, k, E, rows, ldr, None)
    for bad in (dict(x=None), dict(row_of=None), dict(starts=None), dict(rows=None), dict(T=-1), dict(k=0),
                dict(E=0), dict(E=257), dict(dt=-1), dict(d=0), dict(ldr=4), dict(ldx=-8)):
        assert call(**bad) == EINVAL, bad
    assert call(T=0) == _lib.AEM_OK


def test_combine_refusals():
    def call(rows=P, rd=_lib.F32, ldr=8, w=P, ldw=2, row_of=P, T=4, k=2, d=8, out=P, od=_lib.BF16, ldo=8):
        return L().aem_combine(rows, rd, ldr, w, ldw, row_of, T, k, d, out, od, ldo, None)
    for bad in (dict(rows=None), dict(row_of=None), dict(out=None), dict(T=-1), dict(k=0), dict(k=65),
                dict(rd=3), dict(od=3), dict(d=0), dict(ldo=7), dict(ldr=-1), dict(ldw=-1)):
        assert call(**bad) == EINVAL, bad
    assert call(T=0) == _lib.AEM_OK


def test_combine_backward_refusals():
    def call(g=P, gd=_lib.F32, ldg=8, rows=P, rd=_lib.F32, ldr=8, w=P, ldw=2, row_of=P, starts=P, T=4, k=2,
             E=8, d=8, gr=P, ldgr=8, gw=P):
        return L().aem_combine_backward(g, gd, ldg, rows, rd, ldr, w, ldw, row_of, starts, T, k, E, d, gr,
                                        ldgr, gw, None)
    for bad in (dict(g=None), dict(rows=None), dict(row_of=None), dict(starts=None), dict(gr=None, gw=None),
                dict(T=-1), dict(k=0), dict(E=0), dict(gd=9), dict(rd=9), dict(d=0), dict(ldgr=7),
                dict(ldg=-1), dict(ldr=-1), dict(ldw=-1)):
        assert call(**bad) == EINVAL, bad
    assert call(T=0) == _lib.AEM_OK


def test_sort_workspace():
    assert L().aem_token_sort_workspace(0, 2, 8) == 0
    assert L().aem_token_sort_workspace(512, 2, 8) == 0  # at most 1024 units: no scratch
    assert L().aem_token_sort_workspace(513, 2, 8) > 0
    assert L().aem_token_sort_workspace(513, 65, 8) == 0


def test_q4_refusals():
    h = ctypes.c_void_p()
    q = np.zeros((64, 32), np.int8)
    s = np.ones((2, 32), np.float32)

    def pack(q=q, s=s, sd=_lib.F32, G=1, K=64, N=32, gs=32):
        return L().aem_q4weight_pack(None if q is None else q.ctypes.data,
                                     None if s is None else s.ctypes.data, sd, G, K, N, gs, 0,
                                     ctypes.byref(h))
    for bad in (dict(q=None), dict(s=None), dict(sd=5), dict(G=0), dict(K=0), dict(N=0), dict(gs=16),
                dict(gs=48), dict(gs=256)):
        assert pack(**bad) == EINVAL, bad
    wrong = q.copy()
    wrong[5, 7] = 8
    assert pack(q=wrong) == EINVAL and "[-7, 7]" in _lib.last_error()
    wrong[5, 7] = -8
    assert pack(q=wrong) == EINVAL
    if _lib.device_count() == 0:
        assert pack() == _lib.AEM_EUNSUPPORTED
    assert L().aem_quantize_q4(P, _lib.F32, 1, 64, 32, 48, P, P, _lib.F32, None) == EINVAL
    assert L().aem_quantize_q4(P, 4, 1, 64, 32, 64, P, P, _lib.F32, None) == EINVAL
    assert L().aem_quantize_q4(P, _lib.F32, 1, 64, 32, 64, P, P, 4, None) == EINVAL
    assert L().aem_quantize_q4(None, _lib.F32, 1, 64, 32, 64, P, P, _lib.F32, None) == EINVAL
    assert L().aem_quantize_q4(P, _lib.F32, 0, 64, 32, 64, P, P, _lib.F32, None) == EINVAL
    assert L().aem_q4gemm(None, 0, P, _lib.F32, 64, 1, P, _lib.F32, 32, None, 0, None) == EINVAL
    assert L().aem_grouped_q4gemm(None, P, P, _lib.F32, 64, 1, P, _lib.F32, 32, 0, None, 0, None) == EINVAL
    assert L().aem_q4weight_shape(None, None, None, None, None) == EINVAL
    assert L().aem_q4weight_free(None) == _lib.AEM_OK


def test_python_forms_refuse_before_the_library():
    ids = torch.zeros(4, 2, dtype=torch.int32)
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="CUDA"):
        D.dispatch(x, ids, 8)
    with pytest.raises(ValueError, match="int32"):
        D.dispatch(x, ids.long(), 8)
    with pytest.raises(ValueError, match="num_experts"):
        D.sort_tokens(ids, 257)
    with pytest.raises(ValueError, match="k=65"):
        D.sort_tokens(torch.zeros(1, 65, dtype=torch.int32), 128)
    with pytest.raises(ValueError, match="int32"):
        D.TokenOrder(torch.zeros(9), ids, torch.zeros(8, dtype=torch.int32))
    with pytest.raises(ValueError, match="unit_of"):
        D.TokenOrder(torch.zeros(9, dtype=torch.int32), ids, torch.zeros(7, dtype=torch.int32))
    with pytest.raises(ValueError, match="group_size"):
        q4.quantize_q4(torch.zeros(64, 32), 48)
    with pytest.raises(ValueError, match="CUDA"):
        q4.quantize_q4(torch.zeros(64, 32), 32)
    with pytest.raises(ValueError, match="int8"):
        q4.Q4Weight(torch.zeros(64, 32), torch.zeros(2, 32), 32)
    with pytest.raises(ValueError, match="scale must be"):
        q4.Q4Weight(torch.zeros(65, 32, dtype=torch.int8), torch.zeros(2, 32), 32)
    with pytest.raises(ValueError, match="-7, 7"):
        q4.Q4Weight(torch.full((64, 32), 9, dtype=torch.int8), torch.zeros(2, 32), 32)


def test_overlapping_matrices():
    b = torch.zeros(8, 192)
    assert D._overlap(b, b) and D._overlap(b[:, :64], b[:, 63:100]) and D._overlap(b[:, 100:], b[:4, :101])
    assert not D._overlap(b[:, :64], b[:, 64:]) and not D._overlap(b[:, 64:128], b[:, :64])
    assert not D._overlap(b[:4], b[4:]) and D._overlap(b[:5], b[4:])
    assert not D._overlap(b[:0], b) and not D._overlap(b, torch.zeros(8, 192))
    assert D._overlap(b[:1].expand(8, 192), b[1:, :1]) is False and D._overlap(b[:1].expand(8, 192), b)


def test_copies_of_strided_weights_wait_for_the_stream(monkeypatch):
    """A strided weight is copied on the stream that the call was given, so not before
    that stream is entered: a copy on the caller's stream would not be waited for."""
    class Entered(Exception):
        pass

    seen = []

    class Weight(torch.Tensor):
        is_cuda = True

        def contiguous(self, *args, **kwargs):
            seen.append("copied")
            return super().contiguous(*args, **kwargs)

    def enter(stream, fn, tensors, args):
        seen.append("entered")
        raise Entered

    monkeypatch.setattr(q4, "_on", enter)
    w = torch.zeros(32, 64).as_subclass(Weight).t()
    q = torch.zeros(32, 64, dtype=torch.int8).as_subclass(Weight).t()
    scale = torch.ones(32, 2).as_subclass(Weight).t()
    for call in (lambda: q4.quantize_q4(w, 32, stream="side"), lambda: q4.Q4Weight(q, scale, 32, stream="side")):
        with pytest.raises(Entered):
            call()
    assert seen == ["entered", "entered"]


def test_checked_pack_refusals():
    h = ctypes.c_void_p(1)

    def pack(q=P, s=P, sd=_lib.F32, G=1, K=64, N=32, gs=32, out=True):
        return L().aem_q4weight_pack_checked(q, s, sd, G, K, N, gs, None, ctypes.byref(h) if out else None)
    for bad in (dict(q=None), dict(s=None), dict(sd=5), dict(G=0), dict(K=0), dict(N=-1), dict(gs=16)):
        assert pack(**bad) == EINVAL and not h.value, bad
    assert pack(out=False) == EINVAL


def test_gradients_belong_to_the_stream_of_the_call(monkeypatch):
    """The differentiable forms are applied with the given stream current, so autograd
    runs their backward pass there, on the stream that owns the order it reads."""
    seen = []

    class Stream:
        def __init__(self, stream):
            self.stream = stream

        def __enter__(self):
            seen.append(("enter", self.stream))

        def __exit__(self, *args):
            seen.append(("exit", self.stream))

    monkeypatch.setattr(torch.cuda, "stream", Stream)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    for fn in (D._DispatchFn, D._CombineFn):
        monkeypatch.setattr(fn, "apply", lambda *args: seen.append("apply"))
    order = D.TokenOrder(torch.zeros(3, dtype=torch.int32), torch.zeros(4, 2, dtype=torch.int32),
                         torch.zeros(8, dtype=torch.int32))
    x = torch.zeros(4, 8, requires_grad=True)
    for call in (lambda: D.dispatch_rows(x, order, stream="side"),
                 lambda: D.combine(x.new_zeros(8, 8).requires_grad_(), torch.ones(4, 2), order, stream="side")):
        seen.clear()
        call()
        at = seen.index("apply")
        assert seen[at - 1:] == [("enter", "side"), "apply", ("exit", "side")]


def test_forward_mode_is_refused():
    """A dual tensor does not require a gradient, so its tangent would be dropped."""
    from torch.autograd import forward_ad
    order = D.TokenOrder(torch.zeros(3, dtype=torch.int32), torch.zeros(4, 2, dtype=torch.int32),
                         torch.zeros(8, dtype=torch.int32))
    ids = torch.zeros(4, 2, dtype=torch.int32)
    starts = torch.zeros(2, dtype=torch.int32)
    x, rows, w = torch.zeros(4, 8), torch.zeros(8, 8), torch.ones(4, 2)
    with forward_ad.dual_level():
        dx, drows, dw = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, rows, w))
        for call in (lambda: D.dispatch(dx, ids, 2), lambda: D.dispatch_rows(dx, order),
                     lambda: D.combine(drows, w, order), lambda: D.combine(rows, dw, order),
                     lambda: D.combine(drows, None, order), lambda: D.dispatch_backward(drows, order),
                     lambda: D.combine_backward(dx, rows, w, order), lambda: D.combine_backward(x, rows, dw, order),
                     lambda: q4.q4_matmul(dx, None), lambda: q4.grouped_q4_matmul(dx, None, starts)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        with pytest.raises(ValueError, match="CUDA"):  # no tangent: past that check
            D.dispatch(x, ids, 2)
    with pytest.raises(ValueError, match="CUDA"):
        D.dispatch(x, ids, 2)


def test_quantisation_refuses_gradients():
    from torch.autograd import forward_ad
    w = torch.zeros(64, 32, requires_grad=True)
    with pytest.raises(RuntimeError, match="quantize_q4 has no gradient: detach w"):
        q4.quantize_q4(w, 32)
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):  # past that check
        q4.quantize_q4(w, 32)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        q4.quantize_q4(forward_ad.make_dual(w.detach(), torch.ones(64, 32)), 32)


def test_packing_refuses_tensors_of_two_devices():
    """The host pack reads both through their addresses: neither may be a device's."""
    q, s = torch.zeros(64, 32, dtype=torch.int8), torch.ones(2, 32)
    for a, b in ((q, s.to("meta")), (q.to("meta"), s), (q.to("meta"), s.to("meta"))):
        with pytest.raises(ValueError, match="one CUDA device or the CPU"):
            q4.Q4Weight(a, b, 32)


def test_dispatch_backward_refusals():
    def call(g=P, rd=_lib.F32, ldr=8, row_of=P, T=4, k=2, d=8, out=P, xd=_lib.BF16, ldx=8):
        return L().aem_dispatch_backward(g, rd, ldr, row_of, T, k, d, out, xd, ldx, None)
    for bad in (dict(g=None), dict(row_of=None), dict(out=None), dict(T=-1), dict(T=1 << 30), dict(k=0), dict(k=65),
                dict(rd=3), dict(xd=3), dict(d=0), dict(ldx=7), dict(ldr=-1)):
        assert call(**bad) == EINVAL, bad
    assert call(T=0) == _lib.AEM_OK
