"""Argument checks of the routing from logits and of the 8-bit floating point
calls: refused before any GPU work, so they run on any host."""
import ctypes

import pytest
import torch

from aethermoe_b200 import _lib, fp8, routing

P = 4096  # a pointer that no refused call follows
EINVAL = _lib.AEM_EINVAL


def L():
    return _lib.lib()


def config(score=0, k=2, groups=1, top_groups=1, group_top=1, renormalize=0, scale=1.0):
    return ctypes.byref(_lib.RouteConfig(score, k, groups, top_groups, group_top, renormalize, scale))


BAD_CONFIGS = (dict(score=2), dict(k=0), dict(k=65), dict(k=9), dict(groups=0), dict(groups=3), dict(top_groups=0),
               dict(top_groups=2), dict(groups=4, k=3), dict(group_top=0), dict(group_top=3), dict(scale=float("nan")))


def test_route_refusals():
    def call(c=None, x=P, dt=_lib.F32, ld=8, T=4, E=8, ids=P, w=P, **how):
        return L().aem_route_tokens(c or config(**how), x, dt, ld, T, E, None, ids, w, None)
    for bad in BAD_CONFIGS + (dict(x=None), dict(ids=None), dict(w=None), dict(dt=_lib.E4M3), dict(dt=9), dict(ld=-1),
                              dict(T=-1), dict(E=0), dict(E=257), dict(T=1 << 40)):
        assert call(**bad) == EINVAL, bad
    assert call(T=0, x=None) == _lib.AEM_OK
    assert L().aem_route_tokens(None, P, 0, 8, 4, 8, None, P, P, None) == EINVAL


def test_route_backward_refusals():
    def call(g=P, ldg=2, x=P, dt=_lib.F32, ld=8, T=4, E=8, ids=P, ldi=2, out=P, ldo=8, **how):
        return L().aem_route_tokens_backward(config(**how), g, ldg, x, dt, ld, T, E, ids, ldi, out, ldo, None)
    for bad in BAD_CONFIGS + (dict(g=None), dict(x=None), dict(ids=None), dict(out=None), dict(ldo=7), dict(ldg=-1),
                              dict(ldi=-1), dict(dt=3), dict(E=0)):
        assert call(**bad) == EINVAL, bad
    assert call(T=0) == _lib.AEM_OK


def test_quantize_refusals():
    def rows(x=P, dt=_lib.F32, ldx=128, M=4, K=128, q=P, ldq=128, s=P, lds=4):
        return L().aem_quantize_fp8(x, dt, ldx, M, K, q, ldq, s, lds, None)
    for bad in (dict(x=None), dict(q=None), dict(s=None), dict(dt=_lib.E4M3), dict(M=-1), dict(K=0), dict(ldx=-1),
                dict(ldq=127), dict(ldq=112), dict(lds=0), dict(lds=2), dict(K=600), dict(q=P + 8), dict(s=P + 4)):
        assert rows(**bad) == EINVAL, bad
    assert rows(M=0) == _lib.AEM_OK

    def weight(w=P, dt=_lib.F32, G=1, K=64, N=32, q=P, s=P):
        return L().aem_quantize_fp8_weight(w, dt, G, K, N, q, s, None)
    for bad in (dict(w=None), dict(q=None), dict(s=None), dict(dt=2), dict(G=0), dict(K=0), dict(N=0),
                dict(K=1 << 30), dict(G=1 << 20, K=4096, N=4096)):
        assert weight(**bad) == EINVAL, bad


def test_weight_and_product_refusals():
    h = ctypes.c_void_p()
    q, s = torch.zeros(64, 32, dtype=torch.float8_e4m3fn), torch.ones(1, 1)

    def pack(q=q.data_ptr(), s=s.data_ptr(), G=1, K=64, N=32):
        return L().aem_fp8weight_pack(q, s, G, K, N, 0, ctypes.byref(h))
    for bad in (dict(q=None), dict(s=None), dict(G=0), dict(K=0), dict(N=0), dict(N=1 << 30)):
        assert pack(**bad) == EINVAL, bad
    assert L().aem_fp8weight_pack(P, P, 1, 64, 32, 0, None) == EINVAL
    if _lib.device_count() == 0:
        assert pack() == _lib.AEM_EUNSUPPORTED
    assert L().aem_fp8gemm(None, 0, 0, P, 0, 64, None, 0, 1, P, 0, 32, None, 0, None) == EINVAL
    assert L().aem_grouped_fp8gemm(None, P, 0, P, 0, 64, None, 0, 1, P, 0, 32, 0, 0, None, 0, None) == EINVAL
    assert L().aem_fp8weight_shape(None, None, None, None) == EINVAL
    assert L().aem_fp8weight_free(None) == _lib.AEM_OK
    assert L().aem_fp8gemm_workspace(None, 0, 4, 0) == 0


def test_python_forms_refuse_before_the_library():
    x = torch.zeros(4, 8)
    e4m3 = torch.float8_e4m3fn
    with pytest.raises(ValueError, match="CUDA"):
        routing.route_tokens(x, 2)
    with pytest.raises(ValueError, match="softmax"):
        routing.route_tokens(x, 2, score="relu")
    with pytest.raises(RuntimeError, match="no gradient"):
        routing.route_tokens(x, 2, bias=torch.zeros(8, requires_grad=True))
    with pytest.raises(ValueError, match="ids"):
        routing.route_tokens_backward(x, x, torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA"):
        fp8.quantize_fp8(x)
    with pytest.raises(ValueError, match=r"\[K, N\]"):
        fp8.quantize_fp8_weight(torch.zeros(8))
    with pytest.raises(ValueError, match="dtype"):
        fp8.quantize_fp8_weight(torch.zeros(8, 8, dtype=torch.float16))
    with pytest.raises(ValueError, match="float8"):
        fp8.Fp8Weight(torch.zeros(64, 32), torch.ones(1, 1))
    with pytest.raises(ValueError, match="scale must be"):
        fp8.Fp8Weight(torch.zeros(129, 32, dtype=e4m3), torch.ones(1, 1))
    with pytest.raises(ValueError, match="float8"):
        fp8.Fp8Rows(x, torch.ones(4, 1))
    with pytest.raises(ValueError, match="scale must be"):
        fp8.Fp8Rows(x.to(e4m3), torch.ones(4, 2))
    with pytest.raises(RuntimeError, match="forward-mode"):
        import torch.autograd.forward_ad as fwd
        with fwd.dual_level():
            routing.route_tokens(fwd.make_dual(x, x), 2)


def test_readable_rows():
    """Rows that the products can read are taken as they are, others copied."""
    t = torch.zeros(4, 48, dtype=torch.float8_e4m3fn)
    assert fp8._readable(t, 1) == (t, 48)
    assert fp8._readable(t[:, :40], 1)[1] == 48 and fp8._readable(t[:, :40], 1)[0].data_ptr() == t.data_ptr()
    for odd in (t[:, 1:33], t[:, :40].contiguous(), t.t(), t[:, ::2]):
        c, ld = fp8._readable(odd, 1)
        assert ld % 16 == 0 and c.data_ptr() != odd.data_ptr() and torch.equal(c[:, :odd.shape[1]].float(), odd.float())
