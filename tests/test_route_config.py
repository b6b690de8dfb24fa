"""Numbers of a routing configuration that do not fit the C structure are refused
instead of being taken modulo 2^32.  On any host."""
import pytest
import torch

from aethermoe_b200 import routing


@pytest.mark.parametrize("at", [dict(k=2 ** 32 + 2), dict(k=-2 ** 32 + 2), dict(groups=2 ** 32 + 1),
                                dict(groups=2, top_groups=2 ** 33 + 1), dict(groups=2, group_top=2 ** 32 + 2)])
def test_numbers_that_do_not_fit(at):
    with pytest.raises(ValueError, match="out of range"):
        routing.route_tokens(torch.zeros(4, 8), **dict(dict(k=2), **at))
