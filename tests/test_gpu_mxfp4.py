"""MXFP4: quantising, reading back, the product and the product grouped by expert against the format's definition in 64 bits."""
import pytest
import torch

import mxfp4_reference as ref
from nnfusion_amd import ops

pytestmark = pytest.mark.gpu


def _gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen).half()


def _codes(gen, rows, k, low=118, high=131):
    """Any codes, scale bytes of a range, the padding bytes NaN (nobody's arithmetic reads them)."""
    codes = torch.randint(0, 256, (rows, k // 2), generator=gen, dtype=torch.uint8)
    scales = torch.full((rows, ref.scale_bytes(k)), 255, dtype=torch.uint8)
    scales[:, : k // 32] = torch.randint(low, high, (rows, k // 32), generator=gen, dtype=torch.uint8)
    return codes, scales


def _gpu(gpu, *tensors):
    return [None if t is None else t.to(gpu) for t in tensors]


def _equal_bits(a, b):
    return torch.equal(a.cpu().view(torch.int16), b.cpu().view(torch.int16))


# ---- quantising and reading back ---------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("rows,k", [(1, 32), (1, 4096), (3, 64), (5, 480), (7, 512), (2, 544), (33, 1056), (1, 16384), (1000, 2080)])
def test_quantising_is_exact(gpu, rows, k):
    gen = _gen(rows * k)
    x = _normal(gen, rows, k)
    x[:, ::37] *= 40
    codes, scales = ops.mxfp4_quantize(x.to(gpu))
    want_codes, want_scales = ref.quantize(x)
    assert torch.equal(codes.cpu(), want_codes)
    assert torch.equal(scales.cpu(), want_scales)
    assert _equal_bits(ops.mxfp4_dequantize(codes, scales), ref.values(want_codes, want_scales).half())


def test_every_fp16_number_in_a_block_of_its_own_magnitude_and_larger_ones(gpu):
    """All bit patterns, each in blocks whose largest magnitude is their own, 5 and 100 times theirs: ties, subnormals, saturation,
    -0, infinities, NaN."""
    every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.float16)
    x = torch.zeros((65536, 96), dtype=torch.float16)
    for b, factor in enumerate((1.0, 5.0, 100.0)):
        x[:, 32 * b + 7] = every
        x[:, 32 * b + 20] = (every.float() * factor).clamp(-65504, 65504).half() if factor > 1 else every
    codes, scales = ops.mxfp4_quantize(x.to(gpu))
    want_codes, want_scales = ref.quantize(x)
    assert torch.equal(scales.cpu(), want_scales)
    assert torch.equal(codes.cpu(), want_codes)


def test_blocks_of_zeros_and_blocks_that_are_not_finite(gpu):
    x = torch.zeros((4, 128), dtype=torch.float16)
    x[0, 32:64] = 1.0
    x[1, 40] = float("inf")
    x[1, 41] = 3.0
    x[2, 64] = float("nan")
    x[3, 127] = float("-inf")
    x[3, 96] = -0.0
    codes, scales = ops.mxfp4_quantize(x.to(gpu))
    assert scales.cpu()[:, :4].tolist() == [[127, 125, 127, 127], [127, 255, 127, 127], [127, 127, 255, 127], [127, 127, 127, 255]]
    assert not codes.cpu()[1:].any()
    back = ops.mxfp4_dequantize(codes, scales).cpu()
    assert torch.isnan(back[1, 32:64]).all() and torch.isnan(back[2, 64:96]).all() and torch.isnan(back[3, 96:]).all()
    assert int(torch.isnan(back).sum()) == 96


@pytest.mark.parametrize("k", [32, 96, 512, 1024, 1312])
def test_rows_by_index(gpu, k):
    """Rows in another order, several times, not at all; an index that names no row gives zeros."""
    gen = _gen(k)
    x = _normal(gen, 13, k)
    index = torch.tensor([4, 4, 0, 12, -1, 13, 2**31 - 1, -(2**31), 7, 1, 12, 4], dtype=torch.int32)
    codes, scales = ops.mxfp4_quantize(x.to(gpu), rows=index.to(gpu))
    picked = torch.stack([x[i] if 0 <= i < 13 else torch.zeros_like(x[0]) for i in index.tolist()])
    want_codes, want_scales = ref.quantize(picked)
    assert torch.equal(codes.cpu(), want_codes) and torch.equal(scales.cpu(), want_scales)


def test_all_codes_and_all_scale_bytes_are_read_back(gpu):
    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1)  # K = 512: every pair of codes in every row
    scales = torch.arange(256, dtype=torch.uint8)[:, None].repeat(1, 16)
    y = ops.mxfp4_dequantize(*_gpu(gpu, codes, scales)).cpu()
    want = ref.values(codes, scales)
    assert torch.equal(torch.isnan(y), torch.isnan(want))
    fine = ~torch.isnan(want)
    assert _equal_bits(y[fine], want.half()[fine])


def test_given_buffers_are_filled_and_nothing_beside_them(gpu):
    gen = _gen(5)
    x = _normal(gen, 3, 96)
    room_c, room_s = torch.full((5, 48), 0xEE, dtype=torch.uint8, device=gpu), torch.full((5, 16), 0xEE, dtype=torch.uint8, device=gpu)
    codes, scales = ops.mxfp4_quantize(x.to(gpu), codes=room_c[1:4], scales=room_s[1:4])
    want_codes, want_scales = ref.quantize(x)
    assert codes.data_ptr() == room_c[1:4].data_ptr() and scales.data_ptr() == room_s[1:4].data_ptr()
    assert torch.equal(room_c.cpu()[1:4], want_codes) and torch.equal(room_s.cpu()[1:4], want_scales)
    for room in (room_c, room_s):
        assert (room[0] == 0xEE).all() and (room[4] == 0xEE).all()
    room = torch.full((5, 96), 7.0, dtype=torch.float16, device=gpu)
    ops.mxfp4_dequantize(codes.clone(), scales, out=room[1:4])
    assert (room[0] == 7).all() and (room[4] == 7).all() and _equal_bits(room[1:4], ref.values(want_codes, want_scales).half())


# ---- the product -------------------------------------------------------------------------------------------------------------------


def _check(y, want, tol):
    y = y.cpu().double()
    assert torch.isfinite(y).all()
    over = (y - want).abs() > tol
    assert not over.any(), (int(over.sum()), over.nonzero()[:5].tolist(), float(((y - want).abs() / tol).max()))


def _product_case(gpu, gen, m, n, k, bias=False, residual=False, gate=False, variant="auto"):
    a, a_s = _codes(gen, m, k)
    w, w_s = _codes(gen, n * (2 if gate else 1), k, 112, 124)
    b = _normal(gen, n) if bias else None
    r = _normal(gen, m, n) if residual else None
    room = torch.full((m + 2, n), 9.0, dtype=torch.float16, device=gpu) if n % 8 == 0 else None
    out = room[1 : m + 1] if room is not None else None
    ga, gas, gw, gws, gb, gr = _gpu(gpu, a, a_s, w, w_s, b, r)
    y = ops.mxfp4_gemm(ga, gas, gw, gws, bias=gb, residual=gr, act=1 if gate else 0, out=out, variant=variant)
    va, vw = ref.values(a, a_s), ref.values(w, w_s)
    if gate:
        (g, gm), (u, um) = ref.product(va, vw[:n]), ref.product(va, vw[n:])
        want, tol = ref.gated(g, u, gm, um, k)
    else:
        want, magnitude = ref.product(va, vw)
        for more in (b[None, :] if bias else None, r):
            if more is not None:
                want, magnitude = want + more.double(), magnitude + more.double().abs()
        tol = ref.tolerance(want, magnitude, k)
    _check(y, want, tol)
    if room is not None:
        assert (room[0] == 9).all() and (room[m + 1] == 9).all()


ROWS = [1, 2, 15, 16, 17, 31, 33, 64, 65, 100, 128, 129, 200, 257]


@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("n,k", [(64, 512), (100, 1056), (257, 288), (128, 1024)])
def test_product(gpu, m, n, k):
    _product_case(gpu, _gen(m * 1000 + n), m, n, k)


@pytest.mark.parametrize("k", [32, 64, 96, 128, 160, 256, 288, 480, 512, 544, 736, 768, 1024, 1248, 2080, 4096, 11008])
@pytest.mark.parametrize("m", [1, 5, 20, 40, 70, 300])
def test_product_over_k(gpu, m, k):
    _product_case(gpu, _gen(m + k), m, 72, k)


@pytest.mark.parametrize("n", [1, 2, 3, 8, 15, 16, 17, 31, 63, 65, 127, 130, 264, 513])
@pytest.mark.parametrize("m", [1, 18, 50, 140])
def test_product_over_columns(gpu, m, n):
    _product_case(gpu, _gen(m + n), m, n, 416)
    if n < 300:
        _product_case(gpu, _gen(m + n + 1), m, n, 640, gate=True)
        _product_case(gpu, _gen(m + n + 2), m, n, 256, bias=True, residual=True)


@pytest.mark.parametrize("m", [1, 16, 30, 64, 90, 260, 1100, 1300])
def test_epilogues(gpu, m):
    _product_case(gpu, _gen(m), m, 96, 768, bias=True)
    _product_case(gpu, _gen(m + 1), m, 200, 288, residual=True)
    _product_case(gpu, _gen(m + 2), m, 328, 544, bias=True, residual=True)
    _product_case(gpu, _gen(m + 3), m, 144, 1024, gate=True)
    _product_case(gpu, _gen(m + 4), m, 132, 800, gate=True)


@pytest.mark.parametrize("m", [1, 16, 48, 130, 1500])
def test_small_whole_numbers_are_multiplied_exactly(gpu, m):
    """Values 0, +-1, +-2 with scales of 2^0: sums of up to 1024 products of at most 4 are exact in any order, and below 2048 in
    fp16.  Every place of an operand has to meet its partner."""
    gen = _gen(m)
    n, k = 520, 1024
    pick = torch.tensor([0, 2, 4, 10, 12, 0, 0, 0], dtype=torch.uint8)

    def matrix(rows):
        c = pick[torch.randint(0, 8, (rows, k // 2, 2), generator=gen)]
        return c[..., 0] | c[..., 1] << 4, torch.full((rows, ref.scale_bytes(k)), 127, dtype=torch.uint8)

    a, w = matrix(m), matrix(n)
    y = ops.mxfp4_gemm(*_gpu(gpu, *a, *w)).cpu().double()
    want = ref.values(*a) @ ref.values(*w).T
    assert want.abs().max() < 2048
    assert torch.equal(y, want)


@pytest.mark.parametrize("m", [1, 16, 48, 130, 1100])
def test_each_scale_byte_belongs_to_its_block(gpu, m):
    """Ones everywhere, scales 2^0 .. 2^3: sums of whole numbers up to 64 a product, exact, different for any block that takes another's scale."""
    gen = _gen(m)
    n, k = 70, 1056

    def matrix(rows):
        scales = torch.full((rows, ref.scale_bytes(k)), 255, dtype=torch.uint8)
        scales[:, : k // 32] = torch.randint(123, 125, (rows, k // 32), generator=gen, dtype=torch.uint8)
        return torch.full((rows, k // 2), 0x22, dtype=torch.uint8), scales

    a, w = matrix(m), matrix(n)
    y = ops.mxfp4_gemm(*_gpu(gpu, *a, *w)).cpu()
    assert _equal_bits(y, (ref.values(*a) @ ref.values(*w).T).half())


@pytest.mark.parametrize("m", [1, 16, 48, 130, 1100])
def test_not_a_number_stays_in_its_row_and_column(gpu, m):
    gen = _gen(m)
    n, k = 140, 544
    a, a_s = _codes(gen, m, k)
    w, w_s = _codes(gen, n, k)
    a_s[m // 2, 16] = 255
    w_s[77, 3] = 255
    y = torch.isnan(ops.mxfp4_gemm(*_gpu(gpu, a, a_s, w, w_s)).cpu())
    want = torch.zeros((m, n), dtype=torch.bool)
    want[m // 2] = True
    want[:, 77] = True
    assert torch.equal(y, want)


@pytest.mark.parametrize("m", [3, 100])
def test_results_beyond_fp16_are_infinite(gpu, m):
    a = torch.full((m, 128), 0x77, dtype=torch.uint8), torch.full((m, 16), 134, dtype=torch.uint8)
    w = torch.full((16, 128), 0x77, dtype=torch.uint8), torch.full((16, 16), 134, dtype=torch.uint8)
    w[0][8:] = 0xFF
    y = ops.mxfp4_gemm(*_gpu(gpu, *a, *w)).cpu()
    assert (y[:, :8] == float("inf")).all() and (y[:, 8:] == float("-inf")).all()


@pytest.mark.parametrize("m", [2, 40, 150])
def test_the_residual_may_be_the_output(gpu, m):
    gen = _gen(m)
    n, k = 264, 512
    a, a_s = _codes(gen, m, k)
    w, w_s = _codes(gen, n, k, 112, 124)
    r = _normal(gen, m, n)
    ga, gas, gw, gws, gr = _gpu(gpu, a, a_s, w, w_s, r)
    apart = ops.mxfp4_gemm(ga, gas, gw, gws, residual=gr)
    ops.mxfp4_gemm(ga, gas, gw, gws, residual=gr, out=gr)
    assert _equal_bits(apart, gr)


@pytest.mark.parametrize("m,n,k", [(4, 96, 1024), (70, 520, 768), (600, 264, 2048)])
def test_same_call_same_bits(gpu, m, n, k):
    gen = _gen(m)
    operands = _gpu(gpu, *_codes(gen, m, k), *_codes(gen, n, k, 112, 124))
    first = ops.mxfp4_gemm(*operands)
    for _ in range(5):
        assert _equal_bits(first, ops.mxfp4_gemm(*operands))


VARIANTS = [v for v in ops.MXFP4_VARIANTS if v != "auto"]


@pytest.mark.parametrize("variant", VARIANTS)
def test_every_kernel_on_shapes_of_any_size(gpu, variant):
    """Each kernel behind the product: one row and more rows than its tile, columns and K that end inside a tile, a step, a
    pair of steps, a range of K, K shorter than the ranges."""
    for m, n, k in ((1, 1, 32), (7, 40, 64), (9, 33, 96), (16, 64, 256), (17, 70, 288), (33, 130, 512), (65, 129, 544), (130, 260, 1024), (260, 300, 736),
                    (20, 24, 1248), (40, 72, 2080), (3, 56, 4096), (300, 264, 2336), (12, 16, 11008), (8, 104, 8160)):
        _product_case(gpu, _gen(m * 7 + n), m, n, k, bias=n % 2 == 0, residual=m % 2 == 1, variant=variant)
        if ops.mxfp4_variant_supported(variant, 1):
            _product_case(gpu, _gen(m * 7 + n + 1), m, n, k, gate=True, variant=variant)


@pytest.mark.parametrize("variant", VARIANTS)
def test_every_kernel_exactly_and_with_what_is_not_a_number(gpu, variant):
    gen = _gen(31)
    m, n, k = 70, 150, 1056
    pick = torch.tensor([0, 2, 4, 10, 12, 0, 0, 0], dtype=torch.uint8)

    def matrix(rows):
        c = pick[torch.randint(0, 8, (rows, k // 2, 2), generator=gen)]
        scales = torch.full((rows, ref.scale_bytes(k)), 255, dtype=torch.uint8)
        scales[:, : k // 32] = 127
        return c[..., 0] | c[..., 1] << 4, scales

    a, w = matrix(m), matrix(n)
    y = ops.mxfp4_gemm(*_gpu(gpu, *a, *w), variant=variant).cpu().double()
    want = ref.values(*a) @ ref.values(*w).T
    assert want.abs().max() < 2048 and torch.equal(y, want)
    a[1][13, 32] = 255  # the last block
    w[1][149, 0] = 255
    w[1][64, 17] = 255
    y = torch.isnan(ops.mxfp4_gemm(*_gpu(gpu, *a, *w), variant=variant).cpu())
    want = torch.zeros((m, n), dtype=torch.bool)
    want[13], want[:, 149], want[:, 64] = True, True, True
    assert torch.equal(y, want)


@pytest.mark.parametrize("variant", VARIANTS)
def test_every_kernel_grouped(gpu, variant):
    for sizes, n, k in (([1, 0, 3], 40, 96), ([20, 0, 0, 17, 1], 70, 544), ([130, 5, 0, 260], 136, 768), ([0, 0, 9], 33, 2080), ([2] * 70, 24, 256)):
        _grouped_case(gpu, _gen(n), sizes, n, k, first=3, behind=9, variant=variant)
        if ops.mxfp4_variant_supported(variant, 1):
            _grouped_case(gpu, _gen(n + 1), sizes, n, k, gate=True, first=1, behind=70, variant=variant)


@pytest.mark.parametrize("variant", [v for v in ops.MXFP4_VARIANTS if not ops.mxfp4_variant_supported(v, 1)])
def test_kernels_without_a_gate_refuse_it(gpu, variant):
    a, w = _codes(_gen(1), 4, 64), _codes(_gen(2), 32, 64)
    with pytest.raises(ops.NnfError) as e:
        ops.mxfp4_gemm(*_gpu(gpu, *a, *w), act=1, variant=variant)
    assert e.value.status == -2


# ---- grouped by expert -------------------------------------------------------------------------------------------------------------


def _grouped_case(gpu, gen, sizes, n, k, gate=False, first=0, behind=0, variant="auto"):
    experts, rows = len(sizes), n * (2 if gate else 1)
    m = first + sum(sizes) + behind
    a, a_s = _codes(gen, m, k)
    w, w_s = _codes(gen, experts * rows, k, 112, 124)
    w, w_s = w.view(experts, rows, -1), w_s.view(experts, rows, -1)
    at = [first]
    for s in sizes:
        at.append(at[-1] + s)
    out = torch.full((m, n), 5.0, dtype=torch.float16, device=gpu)
    y = ops.mxfp4_grouped_gemm(*_gpu(gpu, a, a_s, w, w_s, torch.tensor(at, dtype=torch.int32)), act=1 if gate else 0, out=out, variant=variant)
    assert y.data_ptr() == out.data_ptr()
    y = y.cpu()
    assert (y[:first] == 5).all() and (y[at[-1] :] == 5).all()
    va = ref.values(a, a_s)
    for e, s in enumerate(sizes):
        if s:
            rows_of = va[at[e] : at[e + 1]]
            vw = ref.values(w[e], w_s[e])
            if gate:
                (g, gm), (u, um) = ref.product(rows_of, vw[:n]), ref.product(rows_of, vw[n:])
                want, tol = ref.gated(g, u, gm, um, k)
            else:
                want, magnitude = ref.product(rows_of, vw)
                tol = ref.tolerance(want, magnitude, k)
            _check(y[at[e] : at[e + 1]], want, tol)


SIZES = [[1], [0, 1], [1, 0, 0], [3, 0, 2, 16, 17], [0, 0, 64, 1], [33, 5, 0, 40], [100, 130, 0, 65], [129, 0, 0, 1, 300], [700, 1, 513], [1, 1, 1, 1, 1, 1, 1000]]


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("n,k,gate", [(64, 512, False), (100, 288, True), (33, 1056, False), (136, 768, True)])
def test_grouped_product(gpu, sizes, n, k, gate):
    _grouped_case(gpu, _gen(sum(sizes) + n), sizes, n, k, gate)


@pytest.mark.parametrize("experts", [63, 64, 65, 130, 300])
def test_many_experts(gpu, experts):
    gen = _gen(experts)
    sizes = torch.randint(0, 4, (experts,), generator=gen).tolist()
    _grouped_case(gpu, gen, sizes, 48, 160, behind=3)
    sizes = [0] * (experts - 1) + [5]
    _grouped_case(gpu, gen, sizes, 40, 96, first=2)


@pytest.mark.parametrize("per_expert", [1, 20, 90, 1100])
def test_rows_outside_the_groups_stay_as_they_are(gpu, per_expert):
    _grouped_case(gpu, _gen(per_expert), [per_expert, 0, per_expert // 2], 72, 256, first=5, behind=70)
    _grouped_case(gpu, _gen(per_expert + 1), [per_expert, 3], 72, 256, gate=True, first=1, behind=1)


@pytest.mark.parametrize("rows", [6, 400])
def test_no_rows_in_any_group(gpu, rows):
    gen = _gen(rows)
    a, a_s = _codes(gen, rows, 64)
    w, w_s = _codes(gen, 3 * 32, 64)
    out = torch.full((rows, 32), 5.0, dtype=torch.float16, device=gpu)
    ops.mxfp4_grouped_gemm(*_gpu(gpu, a, a_s, w.view(3, 32, 32), w_s.view(3, 32, 16), torch.full((4,), 4, dtype=torch.int32)), out=out)
    assert (out == 5).all()


@pytest.mark.parametrize("variant", list(ops.MXFP4_VARIANTS))
@pytest.mark.parametrize("offsets", [[-7, 3, 900, 5], [9, 4, 2, 1], [0, 2**31 - 1, -(2**31), 3], [50, 60, 70, 80], [-5, -4, -3, -2]])
def test_offsets_out_of_order_stay_inside_the_operands(gpu, offsets, variant):
    """What comes out is undefined; rows of Y's neighbours are not touched and the call ends."""
    gen = _gen(1)
    a, a_s = _codes(gen, 20, 64)
    w, w_s = _codes(gen, 3 * 32, 64)
    room = torch.full((60, 32), 5.0, dtype=torch.float16, device=gpu)
    ops.mxfp4_grouped_gemm(*_gpu(gpu, a, a_s, w.view(3, 32, 32), w_s.view(3, 32, 16), torch.tensor(offsets, dtype=torch.int32)), out=room[20:40], variant=variant)
    torch.cuda.synchronize()
    assert (room[:20] == 5).all() and (room[40:] == 5).all()


# ---- together, and as programs use them --------------------------------------------------------------------------------------------


def _mixture(gpu, seed, tokens=37, hidden=256, inter=160, experts=6, top=2):
    gen = _gen(seed)
    x = _normal(gen, tokens, hidden)
    chosen = torch.stack([torch.randperm(experts - 1, generator=gen)[:top] for _ in range(tokens)])  # the last expert gets nothing
    order = torch.argsort(chosen.flatten(), stable=True)
    offsets = torch.cat([torch.zeros(1, dtype=torch.long), torch.bincount(chosen.flatten(), minlength=experts).cumsum(0)]).int()
    up = _codes(gen, experts * 2 * inter, hidden, 114, 122)
    down = _codes(gen, experts * hidden, inter, 114, 122)
    up = up[0].view(experts, 2 * inter, -1), up[1].view(experts, 2 * inter, -1)
    down = down[0].view(experts, hidden, -1), down[1].view(experts, hidden, -1)
    return x, (order // top).int(), offsets, up, down


def test_a_mixture_of_experts(gpu):
    """Tokens in the order of their experts are quantised, go through gate | up with SiLU-gate, are quantised again and go through
    down.  Each call is held to what its own inputs give, so that no step hides another's error."""
    x, token, offsets, up, down = _mixture(gpu, 3)
    gx, gtoken, goffsets = _gpu(gpu, x, token, offsets)
    gup, gdown = _gpu(gpu, *up), _gpu(gpu, *down)
    a, a_s = ops.mxfp4_quantize(gx, rows=gtoken)
    h = ops.mxfp4_grouped_gemm(a, a_s, *gup, goffsets, act=1)
    b, b_s = ops.mxfp4_quantize(h)
    y = ops.mxfp4_grouped_gemm(b, b_s, *gdown, goffsets)
    want = ref.quantize(x[token.long()])
    assert torch.equal(a.cpu(), want[0]) and torch.equal(a_s.cpu(), want[1])
    want = ref.quantize(h.cpu())
    assert torch.equal(b.cpu(), want[0]) and torch.equal(b_s.cpu(), want[1])
    inter = h.shape[1]
    for e in range(offsets.numel() - 1):
        rows = slice(int(offsets[e]), int(offsets[e + 1]))
        if rows.start == rows.stop:
            continue
        va, vw = ref.values(a, a_s)[rows], ref.values(up[0][e], up[1][e])
        (g, gm), (u, um) = ref.product(va, vw[:inter]), ref.product(va, vw[inter:])
        _check(h[rows], *ref.gated(g, u, gm, um, va.shape[1]))
        va, vw = ref.values(b, b_s)[rows], ref.values(down[0][e], down[1][e])
        want, magnitude = ref.product(va, vw)
        _check(y[rows], want, ref.tolerance(want, magnitude, va.shape[1]))


def test_a_layer_after_the_framework_s_normalisation(gpu):
    """RMSNorm -> quantise -> gate | up -> quantise -> down + residual, as the MLP block is put together from these calls."""
    gen = _gen(8)
    m, hidden, inter = 29, 512, 416
    x, gamma = _normal(gen, m, hidden), _normal(gen, hidden)
    up, down = _codes(gen, 2 * inter, hidden, 114, 122), _codes(gen, hidden, inter, 112, 118)
    gx, ggamma, *weights = _gpu(gpu, x, gamma, *up, *down)
    n = ops.rms_norm(gx, ggamma)
    h = ops.mxfp4_gemm(*ops.mxfp4_quantize(n), *weights[:2], act=1)
    y = ops.mxfp4_gemm(*ops.mxfp4_quantize(h), *weights[2:], residual=gx)
    va, vw = ref.values(*ref.quantize(n)), ref.values(*up)
    (g, gm), (u, um) = ref.product(va, vw[:inter]), ref.product(va, vw[inter:])
    _check(h, *ref.gated(g, u, gm, um, hidden))
    va = ref.values(*ref.quantize(h))
    want, magnitude = ref.product(va, ref.values(*down))
    want, magnitude = want + x.double(), magnitude + x.double().abs()
    _check(y, want, ref.tolerance(want, magnitude, inter))


def test_captured_and_replayed(gpu):
    """The whole mixture in a HIP graph, replayed on other inputs and other groups, with eager work between the replays."""
    x, token, offsets, up, down = _mixture(gpu, 11)
    gx, gtoken, goffsets = _gpu(gpu, x, token, offsets)
    gup, gdown = _gpu(gpu, *up), _gpu(gpu, *down)

    def block():
        h = ops.mxfp4_grouped_gemm(*ops.mxfp4_quantize(gx, rows=gtoken), *gup, goffsets, act=1)
        return ops.mxfp4_grouped_gemm(*ops.mxfp4_quantize(h), *gdown, goffsets)

    block()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = block()
    for seed in (21, 22, 23, 24):
        x, token, offsets, _, _ = _mixture(gpu, seed)
        gx.copy_(x), gtoken.copy_(token), goffsets.copy_(offsets)
        eager = block()
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert _equal_bits(y, eager)


def test_two_graphs_and_another_stream_at_once(gpu):
    """Two captured products and an eager one, each on a stream of its own at the same time, give what each gives alone."""
    gen = _gen(4)
    calls = []
    for m, n, k in ((3, 512, 2048), (90, 520, 1024), (300, 264, 768)):
        operands = _gpu(gpu, *_codes(gen, m, k), *_codes(gen, n, k, 112, 124))
        calls.append((operands, ops.mxfp4_gemm(*operands)))
    torch.cuda.synchronize()
    graphs = []
    for operands, _ in calls[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = ops.mxfp4_gemm(*operands)
        graphs.append((graph, y))
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(4):
        for (graph, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            eager = ops.mxfp4_gemm(*calls[2][0])
        torch.cuda.synchronize()
        for got, (_, want) in zip([g[1] for g in graphs] + [eager], calls):
            assert _equal_bits(got, want)


def test_many_rows_and_columns(gpu):
    """A product of several tiles each way, each result against 64 bits."""
    _product_case(gpu, _gen(77), 1300, 1160, 544)
    _product_case(gpu, _gen(78), 1090, 600, 800, gate=True)
