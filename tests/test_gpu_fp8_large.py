"""Block-scaled 8-bit floating point where offsets pass 32 bits and K is the longest there is: what lies at the far end is computed as it is alone."""
import pytest
import torch

import fp8_reference as ref
from nnfusion_amd import ops

pytestmark = pytest.mark.gpu

VARIANTS = [v for v in ops.FP8_VARIANTS if v != "auto"]
F8 = torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def _memory():
    yield
    torch.cuda.empty_cache()


def _gen(gpu, seed):
    g = torch.Generator(device=gpu)
    g.manual_seed(seed)
    return g


def _codes(gpu, gen, *shape):
    """Codes of either sign below 2 in magnitude (filled 2^30 at a time: the generator's own ranges end at 32 bits)"""
    codes = torch.empty(shape, dtype=torch.uint8, device=gpu)
    for part in codes.view(-1).split(1 << 30):
        part.random_(0, 128, generator=gen)
        part.add_(part & 64)  # 0 .. 63, and with the sign 128 .. 191
    return codes.view(F8)


def _scales(gpu, gen, *shape):
    return 0.002 * torch.rand(shape, device=gpu, generator=gen) + 0.001


def _equal_bits(a, b):
    return torch.equal(a.view(torch.int16), b.view(torch.int16))


def test_weights_of_more_than_four_gib(gpu):
    gen = _gen(gpu, 1)
    experts, n, k = 20, 8192, 32768
    w, w_s = _codes(gpu, gen, experts, n, k), _scales(gpu, gen, experts, n // 128, k // 128)
    assert w.numel() > 1 << 32
    a, a_s = _codes(gpu, gen, 24, k), _scales(gpu, gen, k // 128, 24)
    offsets = torch.tensor([0, 2] + [2] * (experts - 2) + [24], dtype=torch.int32, device=gpu)
    alone = a[2:].clone(), a_s[:, 2:].contiguous(), w[-1].clone(), w_s[-1].clone()
    for variant in VARIANTS:
        y = ops.fp8_grouped_gemm(a, a_s, w, w_s, offsets, variant=variant)
        assert torch.isfinite(y).all() and y.abs().max() > 0
        assert _equal_bits(y[2:], ops.fp8_gemm(*alone, variant=variant)), variant
        y = ops.fp8_grouped_gemm(a, a_s, w, w_s, offsets, act=1, variant=variant)  # each expert's rows as gate | up
        assert _equal_bits(y[2:], ops.fp8_gemm(*alone, act=1, variant=variant)), variant


def test_one_matrix_of_more_than_four_gib(gpu):
    gen = _gen(gpu, 6)
    n, k = 140008, 32768
    w, w_s = _codes(gpu, gen, n, k), _scales(gpu, gen, ref.blocks(n), k // 128)
    assert w.numel() > 1 << 32
    a, a_s = _codes(gpu, gen, 3, k), _scales(gpu, gen, k // 128, 3)
    first = n - 300 & ~255  # (the same place in a tile of any width, and in a block of scales)
    for variant in VARIANTS:
        y = ops.fp8_gemm(a, a_s, w, w_s, variant=variant)
        assert _equal_bits(y[:, first:], ops.fp8_gemm(a, a_s, w[first:].clone(), w_s[first // 128 :].clone(), variant=variant)), variant


def test_activations_of_more_than_four_gib(gpu):
    gen = _gen(gpu, 2)
    m, n, k = 140007, 40, 32768
    a, a_s = _codes(gpu, gen, m, k), _scales(gpu, gen, k // 128, m)
    assert a.numel() > 1 << 32
    w, w_s = _codes(gpu, gen, n, k), _scales(gpu, gen, 1, k // 128)
    first = m - 263 & ~255  # (the same place in a tile of any height)
    for variant in VARIANTS:
        y = ops.fp8_gemm(a, a_s, w, w_s, variant=variant)
        assert _equal_bits(y[first:], ops.fp8_gemm(a[first:].clone(), a_s[:, first:].contiguous(), w, w_s, variant=variant)), variant


def test_results_of_more_than_four_gib(gpu):
    gen = _gen(gpu, 3)
    m, n, k = 70001, 32776, 64
    a, a_s = _codes(gpu, gen, m, k), _scales(gpu, gen, 1, m)
    w, w_s = _codes(gpu, gen, n, k), _scales(gpu, gen, ref.blocks(n), 1)
    residual = torch.randn((m, n), device=gpu, dtype=torch.bfloat16, generator=gen)
    first = m - 263 & ~255
    for variant in ("tile_16x32", "tile_64x128", "tile_128x256", "tile_256x256"):
        y = ops.fp8_gemm(a, a_s, w, w_s, residual=residual, variant=variant)
        assert y.numel() * 2 > 1 << 32
        assert _equal_bits(y[first:], ops.fp8_gemm(a[first:].clone(), a_s[:, first:].contiguous(), w, w_s, residual=residual[first:].clone(), variant=variant)), variant
        del y


def test_quantising_more_than_four_gib(gpu):
    rows, k = 300011, 16384
    x = torch.empty((rows, k), device=gpu, dtype=torch.float16)
    gen = _gen(gpu, 4)
    for part in x.split(1 << 15):
        part.normal_(generator=gen)
    assert x.numel() > 1 << 32
    codes, scales = ops.fp8_quantize(x)
    want = ref.quantize(x[-9:])
    assert torch.equal(codes[-9:].view(torch.uint8).cpu(), want[0]) and torch.equal(scales[:, -9:].t().cpu(), want[1])
    index = torch.tensor([rows - 1, 0, rows - 9, rows - 1, rows, -1], dtype=torch.int32, device=gpu)
    picked = ops.fp8_quantize(x, rows=index)
    there = [rows - 1, rows - 9, rows - 1]
    assert torch.equal(picked[0].view(torch.uint8)[[0, 2, 3]], codes.view(torch.uint8)[there]) and torch.equal(picked[1][:, [0, 2, 3]], scales[:, there])
    assert not picked[0][4:].view(torch.uint8).any()
    del codes, scales
    x = x[: rows - 11]  # 300000 rows: matrices of 100000
    codes, scales = ops.fp8_quantize_weights(x.view(3, 100000, k))
    last = 100000 % 128  # the last block's rows
    want = ref.quantize(x[-last:], 128)
    assert torch.equal(codes[2, -last:].view(torch.uint8).cpu(), want[0]) and torch.equal(scales[2, -1:].cpu(), want[1])


@pytest.mark.parametrize("m", [1, 40])
def test_the_longest_rows(gpu, m):
    """K = 2^22, values 0, 1 and -1 and scales of 1: every sum is a whole number below 2^23, so exact in fp32 in any order; one rounding to the result."""
    n, k = 6, 1 << 22
    gen = _gen(gpu, 5)
    pick = torch.tensor([0, 0x38, 0xB8, 0], dtype=torch.uint8, device=gpu)

    def matrix(rows):
        return pick[torch.randint(0, 4, (rows, k), generator=gen, device=gpu)].view(F8)

    a, w = matrix(m), matrix(n)
    a_s, w_s = torch.ones((k // 128, m), device=gpu), torch.ones((1, k // 128), device=gpu)
    wide = w.float()
    want = torch.stack([(a[i].float() * wide).sum(-1) for i in range(m)])  # (whole numbers here too)
    for variant in VARIANTS + ["auto"]:
        assert torch.equal(ops.fp8_gemm(a, a_s, w, w_s, variant=variant), want.half()), variant
        assert torch.equal(ops.fp8_gemm(a, a_s, w, w_s, variant=variant, dtype=torch.bfloat16), want.bfloat16()), variant
    x = a[:2].half()
    codes, scales = ops.fp8_quantize(x)
    assert torch.equal(codes.view(torch.uint8)[:, 64:128].cpu(), ref.quantize(x[:, :128])[0][:, 64:128])
    assert torch.equal(codes.float() * scales.t().repeat_interleave(128, 1), torch.sign(x.float()) * 448 * scales.t().repeat_interleave(128, 1))
