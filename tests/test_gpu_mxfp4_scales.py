"""The scale bytes of the MXFP4 products, kernel by kernel: which block a byte belongs to, bytes at the ends of their range, NaN beside SiLU-gate.
Everything here is exact: the sums are multiples of one unit and below 2^24 of it, so fp32 holds them in whatever order they are
added, and the one rounding to fp16 is that of the exact sum."""
import pytest
import torch

import mxfp4_reference as ref
from nnfusion_amd import ops

pytestmark = pytest.mark.gpu

VARIANTS = list(ops.MXFP4_VARIANTS)
GATED = [v for v in VARIANTS if ops.mxfp4_variant_supported(v, 1)]
# rows and columns that end inside a tile, K that ends inside a step, a pair of steps, a range of K
SHAPES = [(3, 40, 96), (20, 70, 544), (70, 150, 1056), (270, 264, 1376)]


def _gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def _codes(gen, rows, k, pick=range(16)):
    pick = torch.tensor(list(pick), dtype=torch.uint8)
    c = pick[torch.randint(0, len(pick), (rows, k // 2, 2), generator=gen)]
    return c[..., 0] | c[..., 1] << 4


def _scales(rows, k, blocks):
    """blocks: u8 [rows or 1, K/32]; the padding is NaN"""
    s = torch.full((rows, ref.scale_bytes(k)), 255, dtype=torch.uint8)
    s[:, : k // 32] = blocks
    return s


def _random_bytes(gen, rows, k, low, high):
    return torch.randint(low, high, (rows, k // 32), generator=gen, dtype=torch.uint8)


def _equal_bits(a, b):
    return torch.equal(a.cpu().view(torch.int16), b.cpu().view(torch.int16))


def _product(gpu, *operands, **more):
    return ops.mxfp4_gemm(*[t.to(gpu) for t in operands], **more).cpu()


@pytest.mark.parametrize("variant", VARIANTS)
def test_a_scale_byte_belongs_to_the_codes_of_its_block(gpu, variant):
    """Any codes (multiples of 1/2 up to 6), scales 2^-4 .. 2^-1, all drawn: a byte at another block, also one that both operands move alike,
    gives another sum.  Products are multiples of 2^-10 up to 9; 1376 of them stay below 2^24 units."""
    for m, n, k in SHAPES:
        gen = _gen(m + k)
        a, w = ((c, _scales(c.shape[0], k, _random_bytes(gen, c.shape[0], k, 123, 127))) for c in (_codes(gen, m, k), _codes(gen, n, k)))
        want = ref.values(*a) @ ref.values(*w).T
        assert _equal_bits(_product(gpu, *a, *w, variant=variant), want.half()), (m, n, k)
        # the same in groups, the last of them other experts' rows
        half = m // 2
        offsets = torch.tensor([0, half, half, m], dtype=torch.int32)
        w3 = [torch.stack((t, t.flip(0), t.roll(1, 0))) for t in w]
        y = ops.mxfp4_grouped_gemm(*[t.to(gpu) for t in (*a, *w3, offsets)], variant=variant)
        want[half:] = want[half:].roll(1, 1)
        assert _equal_bits(y, want.half()), (m, n, k)


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("extremes", [(0, 254), (1, 253), (254, 0), (253, 1), (0, 1, 2, 126, 128, 252, 253, 254)])
def test_scales_at_both_ends_whose_products_are_ordinary(gpu, variant, extremes):
    """Activations times 2^(x - 127) against weights times 2^(127 - x), x any of the ends from block to block: products of ordinary
    size, multiples of 1/4 up to 36; 416 of them are below 2^24 units."""
    for m, n, k in ((5, 24, 32), (20, 40, 256), (70, 136, 416)):
        gen = _gen(m + sum(extremes))
        x = torch.tensor(extremes, dtype=torch.uint8)[torch.randint(0, len(extremes), (1, k // 32), generator=gen)]
        a, w = _codes(gen, m, k), _codes(gen, n, k)
        y = _product(gpu, a, _scales(m, k, x), w, _scales(n, k, 254 - x), variant=variant)
        one = torch.full((1, k // 32), 127, dtype=torch.uint8)
        assert _equal_bits(y, (ref.values(a, _scales(m, k, one)) @ ref.values(w, _scales(n, k, one)).T).half()), (m, n, k)


@pytest.mark.parametrize("variant", VARIANTS)
def test_products_beyond_fp32_are_zero_or_infinite(gpu, variant):
    """Both scales at one end, signs by row and column: 0 where the products are too small, infinities where they are too large, and 0
    where one of the values is 0, whatever its scale."""
    m, n, k = 40, 72, 544
    gen = _gen(9)
    sign_a, sign_w = torch.randint(0, 2, (m, 1), generator=gen, dtype=torch.uint8), torch.randint(0, 2, (n, 1), generator=gen, dtype=torch.uint8)
    a, w = (c | (s * 0x88) for c, s in ((_codes(gen, m, k, range(1, 8)), sign_a), (_codes(gen, n, k, range(1, 8)), sign_w)))
    a[7] = 0
    w[11] = 0
    ends = lambda rows, byte: _scales(rows, k, torch.full((1, k // 32), byte, dtype=torch.uint8))
    y = _product(gpu, a, ends(m, 0), w, ends(n, 0), variant=variant)
    assert (y == 0).all()
    y = _product(gpu, a, ends(m, 254), w, ends(n, 254), variant=variant)
    want = torch.where((sign_a ^ sign_w.T).bool(), float("-inf"), float("inf")).half()
    want[7], want[:, 11] = 0, 0
    assert torch.equal(y, want)


@pytest.mark.parametrize("variant", GATED)
def test_not_a_number_beside_silu_gate(gpu, variant):
    """A NaN block of a row of activations: the whole row; of a gate row or of an up row: that column.  Nothing else."""
    for m, n, k in SHAPES:
        gen = _gen(m + n)
        a, w = _codes(gen, m, k), _codes(gen, 2 * n, k)
        a_s, w_s = _scales(m, k, _random_bytes(gen, m, k, 118, 123)), _scales(2 * n, k, _random_bytes(gen, 2 * n, k, 114, 120))
        last = k // 32 - 1
        a_s[m // 2, last] = 255
        w_s[n - 1, 0] = 255  # gate
        w_s[n + n // 3, last] = 255  # up
        want = torch.zeros((m, n), dtype=torch.bool)
        want[m // 2], want[:, n - 1], want[:, n // 3] = True, True, True
        assert torch.equal(torch.isnan(_product(gpu, a, a_s, w, w_s, act=1, variant=variant)), want), (m, n, k)
        offsets = torch.tensor([0, m // 2, m], dtype=torch.int32)
        w3, w3_s = torch.stack((w, w)), torch.stack((w_s, w_s))
        w3_s[0, n - 1, 0] = 120  # the first expert's gate is whole
        want[: m // 2, n - 1] = False
        y = ops.mxfp4_grouped_gemm(*[t.to(gpu) for t in (a, a_s, w3, w3_s, offsets)], act=1, variant=variant)
        assert torch.equal(torch.isnan(y.cpu()), want), (m, n, k)
