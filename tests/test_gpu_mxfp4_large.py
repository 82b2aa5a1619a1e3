"""MXFP4 where byte offsets pass 32 bits and K is the longest there is: what lies at the far end is computed as it is alone."""
import pytest
import torch

import mxfp4_reference as ref
from nnfusion_amd import ops

pytestmark = pytest.mark.gpu

VARIANTS = list(ops.MXFP4_VARIANTS)


@pytest.fixture(autouse=True)
def _memory():
    yield
    torch.cuda.empty_cache()


def _codes(gpu, gen, *shape, low=112, high=124):
    *rows, k = shape
    codes = torch.randint(0, 256, (*rows, k // 2), generator=gen, device=gpu, dtype=torch.uint8)
    return codes, torch.randint(low, high, (*rows, ref.scale_bytes(k)), generator=gen, device=gpu, dtype=torch.uint8)


def _gen(gpu, seed):
    g = torch.Generator(device=gpu)
    g.manual_seed(seed)
    return g


def _equal_bits(a, b):
    return torch.equal(a.view(torch.int16), b.view(torch.int16))


def test_weights_of_more_than_four_gib(gpu):
    gen = _gen(gpu, 1)
    experts, n, k = 36, 8192, 32768
    w, w_s = _codes(gpu, gen, experts, n, k)
    assert w.numel() > 1 << 32
    a, a_s = _codes(gpu, gen, 24, k, low=104, high=112)
    offsets = torch.tensor([0, 2] + [2] * (experts - 2) + [24], dtype=torch.int32, device=gpu)
    last = w[-1].clone(), w_s[-1].clone()
    for variant in VARIANTS[1:]:
        y = ops.mxfp4_grouped_gemm(a, a_s, w, w_s, offsets, variant=variant)
        assert torch.isfinite(y).all()
        assert _equal_bits(y[2:], ops.mxfp4_gemm(a[2:].clone(), a_s[2:].clone(), *last, variant=variant)), variant
        if ops.mxfp4_variant_supported(variant, 1):
            y = ops.mxfp4_grouped_gemm(a, a_s, w, w_s, offsets, act=1, variant=variant)
            assert _equal_bits(y[2:], ops.mxfp4_gemm(a[2:].clone(), a_s[2:].clone(), *last, act=1, variant=variant)), variant


def test_activations_of_more_than_four_gib(gpu):
    gen = _gen(gpu, 2)
    m, n, k = 300007, 40, 32768
    a, a_s = _codes(gpu, gen, m, k, low=104, high=112)
    assert a.numel() > 1 << 32
    w, w_s = _codes(gpu, gen, n, k)
    for variant in VARIANTS[1:]:
        y = ops.mxfp4_gemm(a, a_s, w, w_s, variant=variant)
        first = m - 263 & ~255  # (the same place in a tile of any height)
        assert _equal_bits(y[first:], ops.mxfp4_gemm(a[first:].clone(), a_s[first:].clone(), w, w_s, variant=variant)), variant


def test_results_of_more_than_four_gib(gpu):
    gen = _gen(gpu, 3)
    m, n, k = 70001, 32776, 64
    a, a_s = _codes(gpu, gen, m, k)
    w, w_s = _codes(gpu, gen, n, k)
    residual = torch.randn((m, n), device=gpu, dtype=torch.float16, generator=gen)
    for variant in ("auto", "rows_16x32", "tile_64x128", "tile_256x256"):
        y = ops.mxfp4_gemm(a, a_s, w, w_s, residual=residual, variant=variant)
        assert y.numel() * 2 > 1 << 32
        first = m - 263 & ~255
        tail = ops.mxfp4_gemm(a[first:].clone(), a_s[first:].clone(), w, w_s, residual=residual[first:].clone(), variant=variant if variant != "auto" else "tile_256x256")
        va, vw = ref.values(a[first:], a_s[first:]), ref.values(w[-40:], w_s[-40:])
        want, magnitude = ref.product(va, vw)
        more = residual[first:, -40:].cpu().double()
        tol = ref.tolerance(want + more, magnitude + more.abs(), k)
        assert bool(((y[first:, -40:].cpu().double() - want - more).abs() <= tol).all()), variant
        if variant != "auto":
            assert _equal_bits(y[first:], tail), variant
        del y, tail


def test_conversions_of_more_than_four_gib(gpu):
    rows, k = 300011, 8192
    x = torch.randn((rows, k), device=gpu, dtype=torch.float16, generator=_gen(gpu, 4))
    codes, scales = ops.mxfp4_quantize(x)
    far = ops.mxfp4_quantize(x[-9:].clone())
    assert torch.equal(codes[-9:], far[0]) and torch.equal(scales[-9:], far[1])
    want = ref.quantize(x[-9:])
    assert torch.equal(far[0].cpu(), want[0]) and torch.equal(far[1].cpu(), want[1])
    index = torch.tensor([rows - 1, 0, rows - 9, rows - 1, rows, -1], dtype=torch.int32, device=gpu)
    picked = ops.mxfp4_quantize(x, rows=index)
    assert torch.equal(picked[0][[0, 2, 3]], codes[[rows - 1, rows - 9, rows - 1]]) and torch.equal(picked[1][[0, 2, 3]], scales[[rows - 1, rows - 9, rows - 1]])
    assert not picked[0][4:].any() and (picked[1][4:] == 127).all()
    back = ops.mxfp4_dequantize(codes, scales)
    assert torch.equal(back[-9:].cpu().double(), ref.values(codes[-9:], scales[-9:]))  # exact: randn's blocks are far inside fp16


@pytest.mark.parametrize("m", [1, 3, 40])
def test_the_longest_rows(gpu, m):
    """K = 2^22: whole numbers, so that the sums are exact in fp32 in any order; one rounding to fp16."""
    n, k = 6, 1 << 22
    gen = _gen(gpu, 5)
    pick = torch.tensor([0, 2, 10, 0], dtype=torch.uint8, device=gpu)  # 0, 1, -1

    def matrix(rows):
        c = pick[torch.randint(0, 4, (rows, k // 2, 2), generator=gen, device=gpu)]
        return c[..., 0] | c[..., 1] << 4, torch.full((rows, k // 32), 127, dtype=torch.uint8, device=gpu)

    a, w = matrix(m), matrix(n)
    value = torch.tensor([0, 0, 1, 0, 0, 0, 0, 0, 0, 0, -1, 0, 0, 0, 0, 0], dtype=torch.float64, device=gpu)

    def values(codes):
        return torch.stack((value[(codes & 15).long()], value[(codes >> 4).long()]), -1).flatten(-2)

    vw = values(w[0])
    want = torch.stack([(values(a[0][i]) * vw).sum(-1) for i in range(m)]).half()
    for variant in VARIANTS:
        assert torch.equal(ops.mxfp4_gemm(*a, *w, variant=variant), want), variant
    x = torch.stack([values(a[0][i]) for i in range(min(m, 2))]).half()
    codes, scales = ops.mxfp4_quantize(x)
    assert torch.equal(ops.mxfp4_dequantize(codes, scales), x)
