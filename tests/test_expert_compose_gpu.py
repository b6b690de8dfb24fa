"""The expert operators with the framework's own routing, and the C entry points
that Python reaches through another."""
import numpy as np
import pytest

import aem_oracle as O
from test_dispatch_gpu import HALF_BF16, U32, make_ids, plain_order

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,k,E,d", [(1, 2, 8, 16), (200, 2, 8, 24), (600, 6, 64, 40), (3000, 3, 16, 8)])
def test_order_of_capacity_routed_units(cuda, T, k, E, d):
    """The slot-major effective experts of the capacity routing, strides 1 and T, give
    the order of the same experts in a token-major array; a step through it adds up."""
    import torch
    from aethermoe_b200 import _lib
    from aethermoe_b200 import dispatch as D
    rng = np.random.default_rng(T + k)
    idx = make_ids(rng, T, min(k + 1, E), E, "none")
    prim, sec, pos, _, _ = O.moe_units(idx, k, E)
    cap = O.default_capacity(T, k, E)
    want = O.capacity_assign(prim, sec, pos, cap).reshape(k, T).T
    p, s, q = (torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(cuda) for a in (prim, sec, pos))
    eff = torch.empty(k * T, dtype=torch.int32, device=cuda)
    _lib.check(_lib.lib().aem_capacity_route(p.data_ptr(), s.data_ptr(), q.data_ptr(), T * k, E, cap, eff.data_ptr(),
                                             None, 0, torch.cuda.current_stream().cuda_stream))
    ids = eff.view(k, T).t()
    assert ids.stride() == (1, T) or T == 1
    x = torch.from_numpy(rng.integers(-4, 5, size=(T, d)).astype(np.float32)).to(cuda)
    rows, order = D.dispatch(x, ids, E)
    np.testing.assert_array_equal(ids.cpu().numpy(), want)
    starts, row_of, unit_of = plain_order(want, E)
    np.testing.assert_array_equal(order.starts.cpu().numpy(), starts)
    np.testing.assert_array_equal(order.row_of.cpu().numpy(), row_of)
    np.testing.assert_array_equal(order.unit_of.cpu().numpy(), unit_of)
    np.testing.assert_array_equal(rows.cpu().numpy(), x.cpu().numpy()[unit_of // k])
    # whole numbers: the sum of an expert's row times its number is exact
    number = torch.repeat_interleave(torch.arange(1, E + 1, device=cuda), order.starts.diff().long())
    out = D.combine(rows * number[:, None].float(), None, order)
    np.testing.assert_array_equal(out.cpu().numpy(), x.cpu().numpy() * (want + 1).sum(1, keepdims=True))


@pytest.mark.parametrize("rdt,xdt", [("float32", "float32"), ("bfloat16", "bfloat16"), ("float32", "bfloat16"),
                                     ("bfloat16", "float32")])
@pytest.mark.parametrize("T,k,E,d,pad", [(1, 1, 1, 1, 0), (33, 3, 5, 20, 4), (700, 6, 64, 64, 8), (100, 64, 64, 9, 1)])
def test_gradient_of_the_dispatch_in_c(cuda, T, k, E, d, pad, rdt, xdt):
    """``aem_dispatch_backward`` itself, rows of gradients and outputs apart."""
    import torch
    from aethermoe_b200 import _lib
    from aethermoe_b200 import dispatch as D
    rng = np.random.default_rng(T + d)
    rdt, xdt = getattr(torch, rdt), getattr(torch, xdt)
    ids = make_ids(rng, T, k, E, "some")
    order = D.sort_tokens(torch.from_numpy(ids).to(cuda), E)
    _, row_of, _ = plain_order(ids, E)
    g = torch.from_numpy(rng.normal(size=(T * k, d + pad)).astype(np.float32)).to(cuda).to(rdt)
    out = torch.full((T, d + pad), 7.0, device=cuda, dtype=xdt)
    code = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}
    _lib.check(_lib.lib().aem_dispatch_backward(
        g.data_ptr(), code[rdt], d + pad, order.row_of.data_ptr(), T, k, d, out.data_ptr(), code[xdt], d + pad,
        torch.cuda.current_stream().cuda_stream))
    pick = np.where(row_of[:, :, None] >= 0, g.double().cpu().numpy()[np.maximum(row_of, 0)][..., :d], 0.0)
    ref, tol = pick.sum(1), k * U32 * np.abs(pick).sum(1)
    if xdt == torch.bfloat16:
        tol = tol + HALF_BF16 * (np.abs(ref) + tol)
    assert (np.abs(out[:, :d].double().cpu().numpy() - ref) <= tol).all()
    assert (out[:, d:] == 7).all()
    assert torch.equal(out[:, :d], D.dispatch_backward(g[:, :d], order, out_dtype=xdt))
