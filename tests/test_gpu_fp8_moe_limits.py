"""The largest numbers of tokens, rows and matrices that routing and quantising take: whole results against torch's, or what lies at their ends against
the definitions."""
import pytest
import torch

import fp8_reference as ref
from nnfusion_amd import ops

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _memory():
    yield
    torch.cuda.empty_cache()


def _gen(gpu, seed):
    g = torch.Generator(device=gpu)
    g.manual_seed(seed)
    return g


@pytest.mark.parametrize("tokens,n,k", [(1 << 23, 2, 1), (1 << 19, 16, 16), (1 << 20, 300, 8)])
def test_the_most_pairs(gpu, tokens, n, k):
    """2^23 pairs of token and slot.  Logits without equals in a row, so that the order of their sorted values is the choice; weights as in test_gpu_moe:
    within 2^-16 of themselves, here of fp32's softmax, which is as far off again."""
    logits = torch.argsort(torch.rand((tokens, n), device=gpu, generator=_gen(gpu, n)), -1).to(torch.float16)
    weights, experts, rows, offsets, positions = ops.moe_route(logits, k)
    want = logits.float().topk(k, -1)
    assert torch.equal(experts.long(), want.indices)
    score = torch.softmax(logits.float(), -1).gather(-1, want.indices)
    score = score / score.sum(-1, keepdim=True)
    assert bool(((weights - score).abs() <= 2.0 ** -15 * score).all())
    order = torch.sort(want.indices.flatten(), stable=True)
    assert torch.equal(rows.long(), order.indices // k)
    assert torch.equal(positions.flatten().long()[order.indices], torch.arange(tokens * k, device=gpu))
    assert torch.equal(offsets.long(), torch.searchsorted(order.values, torch.arange(n + 1, device=gpu)))


@pytest.mark.parametrize("rows,k", [(1 << 24, 16), (1 << 23, 528)])
def test_the_most_rows_quantised(gpu, rows, k):
    """rows * ceil(K / 512) = 2^24"""
    x = torch.empty((rows, k), dtype=torch.bfloat16, device=gpu)
    gen = _gen(gpu, k)
    for part in x.split(1 << 20):
        part.normal_(generator=gen)
    codes, scales = ops.fp8_quantize(x)
    at = torch.cat([torch.arange(5), torch.randint(0, rows, (40,), generator=torch.Generator().manual_seed(1)), torch.arange(rows - 5, rows)]).to(gpu)
    want = ref.quantize(x[at])
    assert torch.equal(codes.view(torch.uint8)[at].cpu(), want[0]) and torch.equal(scales[:, at].t().cpu(), want[1])
    # and none is missing: a row's largest value is 448 times its scale but for two roundings of fp32, so code 126
    top = codes[:, : min(k, 128)].view(torch.uint8).bitwise_and(127).amax(-1)
    assert bool((top == 126).all())
    del x
    with pytest.raises(RuntimeError):
        ops.fp8_quantize(torch.empty((rows + 1, k), dtype=torch.bfloat16, device=gpu))


def test_the_most_blocks_of_weights(gpu):
    matrices = (1 << 23) - 1
    w = torch.randn((matrices, 1, 16), device=gpu, generator=_gen(gpu, 3)).half()
    codes, scales = ops.fp8_quantize_weights(w)
    want = ref.quantize(w[-50:, 0])
    assert torch.equal(codes.view(torch.uint8)[-50:, 0].cpu(), want[0]) and torch.equal(scales[-50:, 0].cpu(), want[1])
    assert bool((codes.view(torch.uint8).bitwise_and(127).amax(-1) == 126).all())
    with pytest.raises(RuntimeError):
        ops.fp8_quantize_weights(torch.empty((matrices + 1, 1, 16), dtype=torch.float16, device=gpu))
