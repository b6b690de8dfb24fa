"""8-bit values and scales that require a gradient are refused where rows or weights
are made of them: the products have none for them, and autograd would drop it
without a word.  On any host."""
import pytest
import torch

from aethermoe_b200 import fp8

E4M3 = torch.float8_e4m3fn


@pytest.mark.parametrize("make,shape,scale", [(fp8.Fp8Rows, (4, 200), (4, 2)), (fp8.Fp8Weight, (200, 64), (2, 1))])
def test_values_and_scales_with_a_gradient(make, shape, scale):
    leaf = torch.ones(shape, requires_grad=True)
    assert leaf.to(E4M3).requires_grad
    with pytest.raises(RuntimeError, match="no gradient"):
        make(leaf.to(E4M3), torch.ones(scale))
    with pytest.raises(RuntimeError, match="no gradient"):
        make(torch.ones(shape).to(E4M3), torch.ones(scale, requires_grad=True))


def test_allowed_without_gradients():
    q = torch.ones(4, 200, requires_grad=True).to(E4M3)
    with torch.no_grad():
        assert fp8.Fp8Rows(q, torch.ones(4, 2)).shape == (4, 200)
    assert fp8.Fp8Rows(q.detach(), torch.ones(4, 2)).shape == (4, 200)
