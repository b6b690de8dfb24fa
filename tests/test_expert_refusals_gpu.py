"""Refusals of the expert calls that need a GPU to be reached: every one of them
before any work on it."""
import pytest

pytestmark = pytest.mark.gpu


def test_results_of_other_types(cuda):
    """An out of a type that no call writes is refused like an out_dtype of that type."""
    import torch
    from aethermoe_b200 import dispatch as D
    from aethermoe_b200 import fp8, q4
    x = torch.randn(4, 128, device=cuda)
    half = torch.empty(4, 64, device=cuda, dtype=torch.float16)
    starts = torch.tensor([0, 4], device=cuda, dtype=torch.int32)
    w = fp8.Fp8Weight(*fp8.quantize_fp8_weight(torch.randn(1, 128, 64, device=cuda)))
    w4 = q4.Q4Weight(*q4.quantize_q4(torch.randn(1, 128, 64, device=cuda), 64), 64)
    order = D.sort_tokens(torch.zeros(4, 1, device=cuda, dtype=torch.int32), 1)
    for call in (lambda: fp8.fp8_matmul(x, w, out=half), lambda: fp8.fp8_matmul(fp8.quantize_fp8(x), w, out=half),
                 lambda: fp8.grouped_fp8_matmul(x, w, starts, out=half), lambda: q4.q4_matmul(x, w4, out=half),
                 lambda: D.combine(torch.randn(4, 64, device=cuda), None, order, out=half)):
        with pytest.raises(ValueError, match="unsupported dtype"):
            call()
    with pytest.raises(ValueError, match="unsupported dtype"):
        fp8.fp8_matmul(x, w, out_dtype=torch.float16)
