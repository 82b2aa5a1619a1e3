"""Block-scaled 8-bit products whose every partial sum is exact, at long K: a value of K that is lost, counted twice or scaled by another block's scale changes a
result, however long the row.

Codes are 0 and +-1 (one in two), scales 1, 2 for activations and 1/2, 1 for weights, another one in each block: a product is 0 or +-1, eight of them
are alike in size, a block's sum is a whole number up to 128, and what is added is a multiple of 1/2.  A quarter of the products are not zero, with factors of at most 2: a
sum's mean square is at most K (5/2)(5/8) / 4, 98^2 at K = 24592.  Results below 1024 are multiples of 1/2 that fp16 holds: the operands' own test says they are."""
import pytest
import torch

import fp8_reference as ref
from nnfusion_amd import ops

VARIANTS = [v for v in ops.FP8_VARIANTS if v != "auto"]
F8 = torch.float8_e4m3fn
LONG = [8192, 8208, 16400, 16512, 24592]
M, N = 21, 36


def _signs(gen, *shape):
    return (torch.randint(0, 2, shape, generator=gen) * (2 * torch.randint(0, 2, shape, generator=gen) - 1)).double()


def _powers(gen, low, *shape):
    return low * 2.0 ** torch.randint(0, 2, shape, generator=gen).float()


def _operands(m, n, k, experts=None):
    """values [M, K], scales, values [.., N, K], scales"""
    gen, lead = torch.Generator().manual_seed(k + m + n), () if experts is None else (experts,)
    a, w = _signs(gen, m, k), _signs(gen, *lead, n, k)
    # (the last value of K counts in every result)
    a[:, -1], w[..., -1] = 1, 1
    return a, _powers(gen, 1.0, ref.blocks(k), m), w, _powers(gen, 0.5, *lead, ref.blocks(n), ref.blocks(k))


def _sums(a, a_s, w, w_s):
    n, k = w.shape
    return (a * a_s.double().t().repeat_interleave(128, 1)[:, :k]) @ (w * w_s.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]).t()


def _results(a, a_s, w, w_s, dtype=torch.float16):
    return _sums(a, a_s, w, w_s).float().to(dtype)


def _gated(w, w_s, gate_value=None):
    """w as the up rows under gate rows whose sums are all 64 (the first value of a row times 64: SiLU(64) is 64 in fp32), or as gate rows, whose first value gets
    that much more, over up rows whose sums are all 1"""
    n, k = w.shape
    other, other_s = torch.zeros((n, k), dtype=torch.float64), torch.ones_like(w_s)
    if gate_value is None:
        other[:, 0] = 64
        return torch.cat([other, w]), torch.cat([other_s, w_s])
    other[:, 0] = 1
    return torch.cat([w, other]), torch.cat([w_s, other_s])


def _under_gate(k):
    """Operands whose first value is left to the other half of the weight rows"""
    a, a_s, w, w_s = _operands(M, N, k)
    a[:, 0], a_s[0] = 1, 1
    w[:, 0], w_s[:, 0] = 0, 1
    return a, a_s, w, w_s


@pytest.mark.parametrize("k", LONG)
def test_what_the_operands_show(k):
    """On the CPU: results are exact in fp16, and each of these mistakes changes some of them: a row's last value lost, its last 16, one of its
    blocks, or a block's scale: that of the block before for
    activations, the other one of 1/2 and 1 for weights."""
    a, a_s, w, w_s = _operands(M, N, k)
    right = _results(a, a_s, w, w_s)
    assert torch.equal(right.double(), _sums(a, a_s, w, w_s)) and bool((right.abs() < 1024).all())
    assert bool((_sums(*_under_gate(k)).abs() <= 424).all())
    cut = a.clone()
    cut[:, -1] = 0
    assert bool((_results(cut, a_s, w, w_s) != right).all())
    cut[:, -16:] = 0
    assert not torch.equal(_results(cut, a_s, w, w_s), right)
    last = ref.blocks(k) - 1
    for block in {0, 1, 31, 62, 63, 64, 65, 127, 128, last - 1, last}:
        if block > last:
            continue
        cut = a.clone()
        cut[:, block * 128 : block * 128 + 128] = 0
        assert not torch.equal(_results(cut, a_s, w, w_s), right), block
        if block:
            for which, scales in (("a", a_s), ("w", w_s)):
                wrong = scales.clone()
                if which == "a":
                    wrong[block] = wrong[block - 1]
                    assert not torch.equal(_results(a, wrong, w, w_s), right), block
                else:
                    wrong[:, block] = 1.5 - wrong[:, block]
                    assert not torch.equal(_results(a, a_s, w, wrong), right), block


def _on(gpu, a, a_s, w, w_s):
    codes = [t.float().to(F8) for t in (a, w)]
    assert torch.equal(codes[0].double(), a) and torch.equal(codes[1].double(), w)
    return codes[0].to(gpu), a_s.to(gpu), codes[1].to(gpu), w_s.to(gpu)


@pytest.mark.gpu
@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("k", LONG)
def test_long_rows(gpu, variant, k):
    case = _operands(M, N, k)
    on = _on(gpu, *case)
    for dtype in (torch.float16, torch.bfloat16):
        assert torch.equal(ops.fp8_gemm(*on, dtype=dtype, variant=variant).cpu(), _results(*case, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (31, 31, 4096), (130, 300, 656), (257, 130, 1040), (300, 140, 8208), (9, 520, 16512)])
def test_rows_and_columns_of_many_tiles(gpu, variant, m, n, k):
    case = _operands(m, n, k)
    assert torch.equal(ops.fp8_gemm(*_on(gpu, *case), variant=variant).cpu(), _results(*case))


@pytest.mark.gpu
@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("k", [8208, 16512, 24592])
def test_long_rows_with_silu_gate(gpu, variant, k):
    """Through the up rows: 64 times their sums.  Through the gate rows: their sums with 448 added, so at least 24, of which SiLU takes less than 2^-24."""
    a, a_s, w, w_s = _under_gate(k)
    sums = _sums(a, a_s, w, w_s)
    up, up_s = _gated(w, w_s)
    assert torch.equal(ops.fp8_gemm(*_on(gpu, a, a_s, up, up_s), act=1, variant=variant).cpu().double(), 64 * sums)
    lifted = w.clone()
    lifted[:, 0] = 448
    both, both_s = _gated(lifted, w_s, 448)
    assert torch.equal(ops.fp8_gemm(*_on(gpu, a, a_s, both, both_s), act=1, variant=variant).cpu().double(), sums + 448)


@pytest.mark.gpu
@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("k", [8208, 24592])
def test_long_rows_of_groups(gpu, variant, k):
    sizes = [3, 0, 17, 1, 40]
    m, offsets = sum(sizes), torch.tensor([0, 3, 3, 20, 21, 61], dtype=torch.int32)
    a, a_s, w, w_s = _operands(m, N, k, len(sizes))
    y = ops.fp8_grouped_gemm(*_on(gpu, a, a_s, w, w_s), offsets.to(gpu), variant=variant).cpu()
    for e in range(len(sizes)):
        lo, hi = int(offsets[e]), int(offsets[e + 1])
        assert torch.equal(y[lo:hi], _results(a[lo:hi], a_s[:, lo:hi], w[e], w_s[e]))
