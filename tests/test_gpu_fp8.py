"""Block-scaled 8-bit floating point: quantising, the product and the product grouped by expert against the format's definition in 64 bits.

Quantising is exact: codes and scales are what the definition rounds to.  A product: two values' product has eight bits.  The matrix cores add eight of
neighbouring k at a time, each cut, towards zero, to 2^-13 of the power of two of the largest (a single 2^16 beside 1.5 times 2^(16 - e): 2^3 of
2^3 1.5 are left, of 2^2 1.5 nothing, in every one of the other seven places, and all of it in the other places): 8 times 2^-13 of the largest
product, which is at most the product of the largest values.  Then each addition is off by at most a step of fp32 of the magnitudes' sum (2^-23: they may cut);
the scales' product, the product with it and the addition to the sum are off by half a step each, the additions once a block: (130 + blocks)
2^-23 of the sum of magnitudes.  SiLU(g) u: its slope in g is at most
1.1, exp's argument is off by 2^-23 |g|, the rest by a few steps: (|g| + 8) 2^-22.  Then half a step of the result's type, and 2^-25 where fp16 ends."""
import pytest
import torch

import fp8_reference as ref
from nnfusion_amd import _lib, ops

pytestmark = pytest.mark.gpu

VARIANTS = [v for v in ops.FP8_VARIANTS if v != "auto"]
F8 = torch.float8_e4m3fn


def _gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def _codes(gen, *shape):
    """Any finite codes"""
    c = torch.randint(0, 254, shape, generator=gen).to(torch.uint8)
    return torch.where(c >= 127, c + 1, c).view(F8)


def _scales(gen, *shape):
    return torch.exp2(6 * torch.rand(shape, generator=gen) - 8) * (1 + torch.rand(shape, generator=gen))


def _operands(gen, m, n, k, gate=False, experts=None):
    lead, rows, nb = () if experts is None else (experts,), n * (2 if gate else 1), ref.blocks(n) * (2 if gate else 1)
    return _codes(gen, m, k), _scales(gen, ref.blocks(k), m), _codes(gen, *lead, rows, k), 0.02 * _scales(gen, *lead, nb, ref.blocks(k))


def _near(got, want, bound):
    eps = torch.finfo(got.dtype).eps
    got = got.cpu().double()
    limit = bound * (1 + eps) + eps / 2 * want.abs() + 2.0 ** -25
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    off = torch.where(nan, torch.zeros_like(want), got - want).abs()
    assert bool((off <= torch.where(nan, torch.ones_like(limit), limit)).all()), ((off - limit).nan_to_num(-1).max(), off.nan_to_num(0).max())


# ---- quantising -----------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("rows,k", [(1, 16), (1, 4096), (3, 128), (5, 144), (7, 512), (2, 528), (33, 1040), (1, 16384), (1000, 2080), (4099, 1376)])
@pytest.mark.parametrize("type", [torch.float16, torch.bfloat16])
def test_quantised_rows(gpu, rows, k, type):
    gen = _gen(rows + k)
    x = (torch.randn((rows, k), generator=gen) * torch.exp2(16 * torch.rand((rows, 1), generator=gen) - 10)).to(type)
    codes, scales = ops.fp8_quantize(x.to(gpu))
    want, want_scales = ref.quantize(x)
    assert codes.dtype == F8 and torch.equal(scales.cpu(), want_scales.t())
    assert torch.equal(codes.cpu().view(torch.uint8), want)


@pytest.mark.parametrize("type", [torch.float16, torch.bfloat16])
def test_every_value_of_a_type_is_quantised_as_defined(gpu, type):
    """All finite bit patterns, against several largest magnitudes: ties, subnormals, zeros of either sign."""
    bits = torch.arange(0, 1 << 16).to(torch.int16)
    x = bits.view(type)
    x = x[torch.isfinite(x)]
    order = torch.sort(x.abs().double(), stable=True)[1]
    pad = torch.cat([x[order], torch.zeros(-len(x) % 127)]).to(type).view(-1, 127)
    for shift in (0, 1, 5, 12):
        rows = torch.cat([pad, torch.full((len(pad), 1), 0.0).to(type)], 1)
        top = rows.double().abs().amax(1) * 2.0 ** shift * (1 + shift / 7)
        rows[:, 127] = torch.where(top < torch.finfo(type).max, top, 0.0).to(type)
        codes, scales = ops.fp8_quantize(rows.to(gpu))
        want, want_scales = ref.quantize(rows)
        assert torch.equal(scales.cpu(), want_scales.t()) and torch.equal(codes.cpu().view(torch.uint8), want)


def test_ties_after_rounded_scales(gpu):
    """Magnitudes whose scale is not exact and values whose quotient lies at a tie or a step of fp32 beside it."""
    gen = _gen(11)
    top = torch.randint(1024, 2048, (512, 1), generator=gen).double()
    steps = ref.VALUES[1:127]
    between = (steps[:-1] + steps[1:]) / 2
    x = torch.cat([top, (between[torch.randint(0, 125, (512, 127), generator=gen)] * top / 448)], 1)
    for type in (torch.float16, torch.bfloat16):
        codes, scales = ops.fp8_quantize(x.to(type).to(gpu))
        want, want_scales = ref.quantize(x.to(type))
        assert torch.equal(scales.cpu(), want_scales.t()) and torch.equal(codes.cpu().view(torch.uint8), want)


@pytest.mark.parametrize("type", [torch.float16, torch.bfloat16])
def test_quantised_zeros_infinities_and_nan(gpu, type):
    x = torch.randn((4, 400), generator=_gen(1)).to(type)
    x[0, :128] = 0
    x[0, 128:256] = -0.0
    x[1, 130], x[2, 399], x[3, 0] = float("inf"), float("nan"), float("-inf")
    codes, scales = [t.cpu() for t in ops.fp8_quantize(x.to(gpu))]
    want, want_scales = ref.quantize(x)
    assert torch.equal(torch.isnan(scales), torch.isnan(want_scales.t())) and torch.equal(scales.nan_to_num(7), want_scales.t().nan_to_num(7))
    assert torch.equal(codes.view(torch.uint8), want)
    assert bool((scales[0, 0] == 2.0 ** -64 / 448).all()) and torch.isnan(scales).sum() == 3


def test_rows_picked_by_an_index(gpu):
    gen = _gen(3)
    x = torch.randn((50, 272), generator=gen).half()
    index = torch.tensor([3, 3, 49, -1, 50, 0, 2147483647, -2147483648] + torch.randint(0, 50, (300,), generator=gen).tolist(), dtype=torch.int32)
    codes, scales = ops.fp8_quantize(x.to(gpu), rows=index.to(gpu))
    there = (index >= 0) & (index < 50)
    want, want_scales = ref.quantize(torch.where(there[:, None], x[index.clamp(0, 49).long()], torch.zeros_like(x[:1])))
    assert torch.equal(scales.cpu(), want_scales.t()) and torch.equal(codes.cpu().view(torch.uint8), want)
    # (an index that starts on a word only)
    again = ops.fp8_quantize(x.to(gpu), rows=index.to(gpu)[1:])
    assert torch.equal(again[0].view(torch.uint8), codes[1:].view(torch.uint8))


@pytest.mark.parametrize("shape", [(1, 16), (128, 128), (129, 144), (127, 1040), (300, 256), (3, 200, 400), (2, 128, 128), (5, 1, 272), (1, 4099, 2080)])
@pytest.mark.parametrize("type", [torch.float16, torch.bfloat16])
def test_quantised_weights(gpu, shape, type):
    w = torch.randn(shape, generator=_gen(sum(shape))).to(type)
    w.view(-1, shape[-1])[0, 0] = 40
    codes, scales = ops.fp8_quantize_weights(w.to(gpu))
    assert codes.shape == w.shape and codes.dtype == F8 and scales.shape == (*shape[:-2], ref.blocks(shape[-2]), ref.blocks(shape[-1]))
    for i, matrix in enumerate(w.view(-1, *shape[-2:])):
        want, want_scales = ref.quantize(matrix, 128)
        assert torch.equal(codes.view(torch.uint8).view(-1, *shape[-2:])[i].cpu(), want)
        assert torch.equal(scales.view(-1, *scales.shape[-2:])[i].cpu(), want_scales)


def test_quantised_into_the_caller_s_buffers_and_nowhere_else(gpu):
    x = torch.randn((37, 176), generator=_gen(6)).half().to(gpu)
    for what in ("rows", "weights"):
        nb = (2, 37) if what == "rows" else (1, 2)
        guarded = torch.full((64 + 37 * 176 + 64,), 9, dtype=torch.uint8, device=gpu), torch.full((8 + nb[0] * nb[1] + 8,), 9.0, device=gpu)
        codes, scales = guarded[0][64:-64].view(F8).view(37, 176), guarded[1][8:-8].view(*nb)
        call = (lambda **kw: ops.fp8_quantize(x, **kw)) if what == "rows" else (lambda **kw: ops.fp8_quantize_weights(x, **kw))
        got, want = call(codes=codes, scales=scales), call()
        assert got[0] is codes and got[1] is scales
        assert torch.equal(codes.view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(scales, want[1])
        for g, edge in zip(guarded, (64, 8)):
            assert bool((g[:edge] == 9).all()) and bool((g[-edge:] == 9).all())


# ---- the product ----------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (1, 128, 128), (3, 5, 144), (17, 33, 272), (16, 200, 1040), (33, 130, 528), (64, 64, 1536), (65, 257, 656), (130, 129, 2064),
                                   (257, 300, 1280), (5, 40, 16400), (31, 31, 4096)])
@pytest.mark.parametrize("type", [torch.float16, torch.bfloat16])
def test_products(gpu, variant, m, n, k, type):
    a, a_s, w, w_s = _operands(_gen(m + n + k), m, n, k)
    y = ops.fp8_gemm(a.to(gpu), a_s.to(gpu), w.to(gpu), w_s.to(gpu), dtype=type, variant=variant)
    assert y.dtype == type
    _near(y, *ref.product(ref.row_values(a, a_s), ref.weight_values(w, w_s, n), n))


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (2, 128, 256), (19, 40, 400), (64, 136, 1040), (70, 65, 528), (200, 300, 912), (33, 16, 2064)])
def test_silu_gate(gpu, variant, m, n, k):
    a, a_s, w, w_s = _operands(_gen(m * n + k), m, n, k, gate=True)
    y = ops.fp8_gemm(a.to(gpu), a_s.to(gpu), w.to(gpu), 1e-3 * w_s.to(gpu), act=1, variant=variant)
    _near(y, *ref.product(ref.row_values(a, a_s), ref.weight_values(w, 1e-3 * w_s, n), n, gate=True))


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("m,n,k", [(1, 8, 128), (45, 67, 272), (130, 256, 384), (7, 130, 144)])
@pytest.mark.parametrize("type", [torch.float16, torch.bfloat16])
def test_bias_and_residual(gpu, variant, m, n, k, type):
    gen = _gen(m + n)
    a, a_s, w, w_s = _operands(gen, m, n, k)
    bias, residual = torch.randn((n,), generator=gen).to(type), torch.randn((m, n), generator=gen).to(type)
    on = [t.to(gpu) for t in (a, a_s, w, w_s)]
    av, wv = ref.row_values(a, a_s), ref.weight_values(w, w_s, n)
    for b, r in ((bias, None), (None, residual), (bias, residual)):
        y = ops.fp8_gemm(*on, bias=None if b is None else b.to(gpu), residual=None if r is None else r.to(gpu), variant=variant)
        assert y.dtype == type
        _near(y, *ref.product(av, wv, n, bias=b, residual=r))
    # the residual as the output
    y = residual.to(gpu)
    got = ops.fp8_gemm(*on, bias=bias.to(gpu), residual=y, out=y, variant=variant)
    assert got is y and torch.equal(y, ops.fp8_gemm(*on, bias=bias.to(gpu), residual=residual.to(gpu), variant=variant))


@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (16, 11008, 1376), (300, 1030, 2064), (2048, 640, 512), (4, 70000, 256)])
def test_products_of_the_library_s_choice(gpu, m, n, k):
    a, a_s, w, w_s = _operands(_gen(m + n + k), m, n, k)
    _near(ops.fp8_gemm(a.to(gpu), a_s.to(gpu), w.to(gpu), w_s.to(gpu)), *ref.product(ref.row_values(a, a_s), ref.weight_values(w, w_s, n), n))


@pytest.mark.parametrize("variant", VARIANTS)
def test_rows_and_columns_do_not_touch_each_other(gpu, variant):
    """NaN codes and scales, infinite scales and zero scales: only what they belong to changes."""
    gen = _gen(9)
    m, n, k = 70, 260, 656
    a, a_s, w, w_s = _operands(gen, m, n, k)
    plain = ops.fp8_gemm(*[t.to(gpu) for t in (a, a_s, w, w_s)], variant=variant).cpu()
    a2, a_s2, w2, w_s2 = a.clone().view(torch.uint8), a_s.clone(), w.clone().view(torch.uint8), w_s.clone()
    a2[3, 655], a2[68, 0], w2[259, 650], w2[100, 130] = 0x7F, 0xFF, 0x7F, 0xFF
    a_s2[2, 10], a_s2[5, 11], w_s2[1, 4] = float("nan"), float("inf"), float("nan")
    y = ops.fp8_gemm(a2.view(F8).to(gpu), a_s2.to(gpu), w2.view(F8).to(gpu), w_s2.to(gpu), variant=variant).cpu()
    rows, columns = torch.zeros(m, dtype=torch.bool), torch.zeros(n, dtype=torch.bool)
    rows[[3, 68, 10, 11]] = True
    columns[[259, 100]] = True
    columns[128:256] = True
    fine = ~rows[:, None] & ~columns[None, :]
    assert torch.equal(y[fine].view(torch.int16), plain[fine].view(torch.int16))
    assert bool(torch.isnan(y[[3, 68, 10]]).all()) and bool(torch.isnan(y[:, columns]).all()) and not bool(torch.isfinite(y[11]).any())


def test_scales_of_each_block_are_used(gpu):
    """One block of K at a time has scales other than zero."""
    m, n, k = 40, 300, 1040
    a, a_s, w, w_s = _operands(_gen(2), m, n, k)
    for b in range(ref.blocks(k)):
        only = torch.zeros_like(a_s)
        only[b] = a_s[b]
        for variant in VARIANTS:
            y = ops.fp8_gemm(a.to(gpu), only.to(gpu), w.to(gpu), w_s.to(gpu), variant=variant)
            _near(y, *ref.product(ref.row_values(a, only), ref.weight_values(w, w_s, n), n))


@pytest.mark.parametrize("variant", VARIANTS)
def test_more_than_64_blocks_of_k(gpu, variant):
    for k in (8192, 8208, 16384 + 128, 3 * 8192 + 16):
        a, a_s, w, w_s = _operands(_gen(k), 5, 36, k)
        _near(ops.fp8_gemm(a.to(gpu), a_s.to(gpu), w.to(gpu), w_s.to(gpu), variant=variant), *ref.product(ref.row_values(a, a_s), ref.weight_values(w, w_s, 36), 36))


@pytest.mark.parametrize("variant", VARIANTS)
def test_results_stay_inside_the_output(gpu, variant):
    for m, n in ((33, 100), (5, 7), (130, 264)):
        a, a_s, w, w_s = [t.to(gpu) for t in _operands(_gen(m), m, n, 272)]
        guarded = torch.full((64 + m * n + 64,), 7.0, dtype=torch.float16, device=gpu)
        out = guarded[64:-64].view(m, n)
        assert torch.equal(ops.fp8_gemm(a, a_s, w, w_s, out=out, variant=variant), ops.fp8_gemm(a, a_s, w, w_s, variant=variant))
        assert bool((guarded[:64] == 7).all()) and bool((guarded[-64:] == 7).all())


# ---- grouped by expert -----------------------------------------------------------------------------------------------------------------


def _check_grouped(gpu, sizes, n, k, gate, variant, first=0, pad=0, type=torch.float16):
    experts, m = len(sizes), first + sum(sizes) + pad
    a, a_s, w, w_s = _operands(_gen(m + n + k), m, n, k, gate, experts)
    if gate:
        w_s = 1e-3 * w_s
    offsets = torch.tensor([first] + [first + sum(sizes[: i + 1]) for i in range(experts)], dtype=torch.int32)
    out = torch.full((m, n), 7.0, dtype=type, device=gpu)
    got = ops.fp8_grouped_gemm(a.to(gpu), a_s.to(gpu), w.to(gpu), w_s.to(gpu), offsets.to(gpu), act=1 if gate else 0, out=out, variant=variant)
    assert got is out
    av, wv = ref.row_values(a, a_s), ref.weight_values(w, w_s, n)
    for e in range(experts):
        lo, hi = int(offsets[e]), int(offsets[e + 1])
        if hi > lo:
            _near(out[lo:hi], *ref.product(av[lo:hi], wv[e], n, gate))
    assert bool((out[:first] == 7).all()) and bool((out[first + sum(sizes):] == 7).all())


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("sizes,n,k", [([1], 32, 128), ([0, 5, 0, 17, 1, 0], 65, 272), ([130, 0, 3, 64, 33], 136, 400), ([2] * 70, 24, 144), ([0, 0, 9], 128, 256)])
def test_grouped_products(gpu, variant, gate, sizes, n, k):
    _check_grouped(gpu, sizes, n, k, gate, variant)


@pytest.mark.parametrize("variant", VARIANTS + ["auto"])
def test_rows_of_no_group_are_left_as_they_are(gpu, variant):
    _check_grouped(gpu, [3, 0, 40, 1], 70, 272, False, variant, first=5, pad=77)
    _check_grouped(gpu, [0, 0], 70, 272, True, variant, first=3, pad=4, type=torch.bfloat16)


def test_a_group_of_its_own_is_the_plain_product(gpu):
    a, a_s, w, w_s = [t.to(gpu) for t in _operands(_gen(4), 100, 200, 528, experts=1)]
    offsets = torch.tensor([0, 100], dtype=torch.int32, device=gpu)
    for variant in VARIANTS:
        assert torch.equal(ops.fp8_grouped_gemm(a, a_s, w, w_s, offsets, variant=variant), ops.fp8_gemm(a, a_s, w[0], w_s[0], variant=variant))


def test_offsets_that_break_their_promise_stay_inside(gpu):
    """Falling, negative and too large offsets: undefined rows of Y, nothing else."""
    m, n, k, experts = 60, 40, 144, 5
    a, a_s, w, w_s = [t.to(gpu) for t in _operands(_gen(4), m, n, k, experts=experts)]
    for bad in ([0, 50, 10, 60, 20, 60], [-5, 3, 1000, 60, -1, 70], [60, 50, 40, 30, 20, 10], [2147483647, -2147483648, 0, 60, 60, 60]):
        for variant in VARIANTS:
            guarded = torch.full((64 + m * n + 64,), 7.0, dtype=torch.float16, device=gpu)
            ops.fp8_grouped_gemm(a, a_s, w, w_s, torch.tensor(bad, dtype=torch.int32, device=gpu), out=guarded[64:-64].view(m, n), variant=variant)
            assert bool((guarded[:64] == 7).all()) and bool((guarded[-64:] == 7).all())


def test_captured_and_replayed(gpu):
    gen = _gen(12)
    x = torch.zeros((40, 400), dtype=torch.bfloat16, device=gpu)
    w = torch.randn((3, 72, 400), generator=gen).bfloat16().to(gpu)
    offsets = torch.zeros(4, dtype=torch.int32, device=gpu)
    wq, ws = ops.fp8_quantize_weights(w)
    y = torch.full((40, 72), 7.0, dtype=torch.bfloat16, device=gpu)

    def step(out):
        a, a_s = ops.fp8_quantize(x)
        return ops.fp8_grouped_gemm(a, a_s, wq, ws, offsets, out=out), ops.fp8_gemm(a, a_s, wq[0], ws[0], dtype=torch.bfloat16)

    step(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, dense = step(y)
    for seed, ends in ((1, [0, 7, 7, 40]), (2, [0, 0, 0, 0]), (3, [0, 1, 39, 40])):
        x.copy_(torch.randn((40, 400), generator=_gen(seed)))
        offsets.copy_(torch.tensor(ends, dtype=torch.int32))
        y.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        want = torch.full_like(y, 7)
        _, want_dense = step(want)
        assert torch.equal(y, want) and torch.equal(dense, want_dense)


def test_on_another_stream(gpu):
    a, a_s, w, w_s = [t.to(gpu) for t in _operands(_gen(4), 100, 200, 528)]
    want = ops.fp8_gemm(a, a_s, w, w_s)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = ops.fp8_gemm(a, a_s, w, w_s)
    stream.synchronize()
    assert torch.equal(got, want)


# ---- together -------------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("tokens,live", [(1, None), (37, None), (200, 150)])
def test_a_mixture_of_experts(gpu, tokens, live):
    """Routing, quantising in the experts' order, gate and up, quantising, down, combining: each step against the one before it as it came out."""
    import moe_reference as moe

    gen = _gen(tokens)
    experts, k, h, i = 12, 3, 272, 200
    x, logits, bias = torch.randn((tokens, h), generator=gen).bfloat16(), torch.randn((tokens, experts), generator=gen), 0.1 * torch.randn((experts,), generator=gen)
    wgu, wd = (torch.randn((2 * experts, i, h), generator=gen) / h ** 0.5).bfloat16(), (torch.randn((experts, h, i + 8), generator=gen) / i ** 0.5).bfloat16()
    wd[:, :, i:] = 0  # (rows of a multiple of 16)
    count = None if live is None else torch.tensor([live], dtype=torch.int32, device=gpu)
    there = tokens if live is None else live
    gu, gu_s = ops.fp8_quantize_weights(wgu.to(gpu))
    gu, gu_s = gu.view(experts, 2 * i, h), gu_s.view(experts, -1, gu_s.shape[-1])
    d, d_s = ops.fp8_quantize_weights(wd.to(gpu))

    weights, ids, rows, offsets, positions = ops.moe_route(logits.to(gpu), k, score="sigmoid", bias=bias.to(gpu), groups=4, top_groups=2, group_top=2, tokens=count)
    a, a_s = ops.fp8_quantize(x.to(gpu), rows=rows)
    hidden = ops.fp8_grouped_gemm(a, a_s, gu, gu_s, offsets, act=1, out=torch.zeros((tokens * k, i), dtype=torch.bfloat16, device=gpu))
    padded = torch.zeros((tokens * k, i + 8), dtype=torch.bfloat16, device=gpu)
    padded[:, :i] = hidden
    b, b_s = ops.fp8_quantize(padded)
    y = ops.fp8_grouped_gemm(b, b_s, d, d_s, offsets, out=torch.full((tokens * k, h), float("nan"), dtype=torch.bfloat16, device=gpu))
    out = ops.moe_combine(y, weights, positions, residual=x.to(gpu))

    want = moe.route(logits, k, score="sigmoid", bias=bias, groups=4, top_groups=2, group_top=2, tokens=live)
    for got, w in zip((ids, rows, offsets, positions), want[1:]):
        assert torch.equal(got.cpu(), w)
    picked = torch.where((rows.cpu() >= 0)[:, None], x[rows.cpu().clamp(min=0).long()], torch.zeros_like(x[:1]))
    codes, scales = ref.quantize(picked)
    assert torch.equal(a.cpu().view(torch.uint8), codes) and torch.equal(a_s.cpu(), scales.t())
    av, guv, bv, dv = ref.row_values(a, a_s), ref.weight_values(gu, gu_s, i), ref.row_values(b, b_s), ref.weight_values(d, d_s, h)
    for e in range(experts):
        lo, hi = int(offsets[e]), int(offsets[e + 1])
        if hi > lo:
            _near(hidden[lo:hi], *ref.product(av[lo:hi], guv[e], i, gate=True))
            _near(y[lo:hi], *ref.product(bv[lo:hi], dv[e], h))
    want_out, size = moe.combine(y, weights, positions, x)
    assert bool(((out.cpu().double() - want_out).abs() <= 2.0 ** -8 * want_out.abs() + (k + 2) * 2.0 ** -23 * size).all())
    assert torch.equal(out[there:].cpu(), x[there:])


def test_route_with_the_mxfp4_products(gpu):
    gen = _gen(21)
    x, logits = torch.randn((30, 256), generator=gen).half().to(gpu), torch.randn((30, 8), generator=gen).to(gpu)
    w = torch.randn((8 * 96, 256), generator=gen).half().to(gpu)
    wq, ws = ops.mxfp4_quantize(w)
    weights, ids, rows, offsets, positions = ops.moe_route(logits, 2)
    a, a_s = ops.mxfp4_quantize(x, rows=rows)
    y = ops.moe_combine(ops.mxfp4_grouped_gemm(a, a_s, wq.view(8, 96, -1), ws.view(8, 96, -1), offsets), weights, positions)
    for t in (0, 7, 29):
        row = sum(weights[t, j] * ops.mxfp4_gemm(*ops.mxfp4_quantize(x[t:t + 1].contiguous()), wq.view(8, 96, -1)[ids[t, j]], ws.view(8, 96, -1)[ids[t, j]]).float() for j in range(2))
        # two roundings of the experts' rows in fp16 either way (other kernels, another order of sums: a step), one of the result
        assert bool(((y[t].float() - row[0]).abs() <= 2.0 ** -9 * row[0].abs() + 2.0 ** -9 * 2 * 64).all())


def test_nothing_to_do_is_refused(gpu):
    x, w, no = torch.zeros((0, 256), dtype=torch.float16, device=gpu), torch.zeros((8, 256), dtype=torch.float16, device=gpu), torch.zeros(0, dtype=torch.int32, device=gpu)
    wq, ws = ops.fp8_quantize_weights(w)
    a, a_s = ops.fp8_quantize(w)
    for call in (lambda: ops.fp8_quantize(x), lambda: ops.fp8_quantize(w, rows=no), lambda: ops.fp8_quantize_weights(x), lambda: ops.fp8_gemm(a[:0], a_s[:, :0], wq, ws),
                 lambda: ops.fp8_gemm(a, a_s, wq[:0], ws[:0]), lambda: ops.fp8_grouped_gemm(a, a_s, wq[None][:0], ws[None][:0], torch.zeros(1, dtype=torch.int32, device=gpu))):
        with pytest.raises(RuntimeError):
            call()
