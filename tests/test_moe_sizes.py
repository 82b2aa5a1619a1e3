"""Sizes that routing does not serve: the workspace query gives 0 for them, and the front refuses them ahead of making their results."""
import pytest
import torch

from nnfusion_amd import ops

MOST = 1 << 23  # pairs of token and slot


@pytest.mark.parametrize("tokens,experts,k", [(2147483647, 256, 8), (2147483647, 1024, 1), (1 << 24, 256, 8), (MOST + 1, 2, 1), ((MOST >> 3) + 1, 256, 8), (2147483647, 256, 2147483647),
                                              (1000, 1025, 8), (1000, 2147483647, 8), (1000, 256, 17), (1000, 256, 0), (1000, 256, -1), (-5, 256, 8), (1000, -1, 8), (0, 256, 8)])
def test_no_workspace_for_sizes_that_are_not_served(tokens, experts, k):
    assert ops.moe_route_workspace_bytes(tokens, experts, k) == 0


@pytest.mark.parametrize("tokens,experts,k", [(MOST, 1024, 1), (MOST >> 4, 1024, 16), (17, 256, 16), (9, 257, 1)])
def test_the_workspace_of_what_is_served(tokens, experts, k):
    """A row of 16-bit counts for each of up to 256 workgroups."""
    need = ops.moe_route_workspace_bytes(tokens, experts, k)
    assert 0 < need <= 256 * ((experts + 1) // 2) * 4


@pytest.mark.parametrize("tokens,experts,k", [(MOST + 1, 1, 1), (MOST // 8 + 1, 8, 8)])
def test_too_many_pairs_are_refused_ahead_of_their_results(tokens, experts, k):
    """On host tensors, whose results no call makes: what is said is not that they lie on the host."""
    with pytest.raises(ops.NnfError) as error:
        ops.moe_route(torch.empty((tokens, experts)), k)
    assert error.value.status == -2
