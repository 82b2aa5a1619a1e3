"""Combining onto a residual that is the result's own memory, with rows that start on 16 bytes and rows that do not."""
import pytest
import torch

import moe_reference as ref
from nnfusion_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,k,n", [(1, 1, 1), (7, 3, 61), (33, 2, 513), (5, 9, 4099), (64, 8, 4096), (300, 16, 1030)])
@pytest.mark.parametrize("type", [torch.float16, torch.bfloat16])
def test_onto_itself(gpu, tokens, k, n, type):
    gen = torch.Generator().manual_seed(tokens + n)
    x, residual = torch.randn((tokens * k, n), generator=gen).to(type), torch.randn((tokens, n), generator=gen).to(type)
    weights, positions = torch.rand((tokens, k), generator=gen), torch.randperm(tokens * k, generator=gen).int().view(tokens, k)
    on = [t.to(gpu) for t in (x, weights, positions)]
    y = residual.to(gpu)
    assert ops.moe_combine(*on, y, y) is y
    assert torch.equal(y, ops.moe_combine(*on, residual.to(gpu)))
    # a product and an addition for each term, half a step of the result; 2^-25 where fp16 ends
    want, size = ref.combine(x, weights, positions, residual)
    eps = torch.finfo(type).eps
    assert bool(((y.cpu().double() - want).abs() <= eps / 2 * want.abs() + (k + 2) * 2.0 ** -24 * size * (1 + eps) + 2.0 ** -25).all())
