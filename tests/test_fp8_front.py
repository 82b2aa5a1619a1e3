"""What the calls on block-scaled 8-bit floating point refuse, on host tensors and at the C entry points: nothing here reaches a kernel."""
import pytest
import torch

from nnfusion_amd import _lib, ops

INVALID, UNSUPPORTED, NO_DEVICE = -1, -2, -4
F8, HALF = torch.float8_e4m3fn, torch.float16


def _f8(*shape):
    return torch.zeros(shape, dtype=torch.uint8).view(F8)


def _strided(t):
    return t.view(torch.uint8).repeat_interleave(2, -1)[..., ::2].view(F8) if t.dtype == F8 else t.repeat_interleave(2, -1)[..., ::2]


def _refused(function, good, bad):
    for what, change in bad.items():
        with pytest.raises(AssertionError):
            function(**{**good, **change})
            pytest.fail(what)


def test_quantising_refuses_what_it_would_misread():
    x = torch.zeros((4, 272), dtype=HALF)
    index = torch.zeros(3, dtype=torch.int32)
    _refused(ops.fp8_quantize, {"x": x}, {
        "fp32": {"x": x.float()}, "strided": {"x": _strided(x)}, "int64 rows": {"rows": index.long()}, "rows of two axes": {"rows": index[None]},
        "strided rows": {"rows": torch.zeros(6, dtype=torch.int32)[::2]}, "codes of bytes": {"codes": torch.zeros((4, 272), dtype=torch.uint8)},
        "codes of fewer rows": {"codes": _f8(3, 272)}, "codes of x's rows, not of the index": {"rows": index, "codes": _f8(4, 272)},
        "scales a row": {"scales": torch.zeros((4, 3))}, "fp16 scales": {"scales": torch.zeros((3, 4), dtype=HALF)}, "fewer scales": {"scales": torch.zeros((2, 4))},
        "strided codes": {"codes": _strided(_f8(4, 272))}, "host tensors": {},
    })
    for args, error in (((x[0],), ValueError), ((None,), TypeError), ((x.numpy(),), TypeError), ((x, [0, 1]), TypeError)):
        with pytest.raises(error):
            ops.fp8_quantize(*args)


def test_quantising_weights_refuses_what_it_would_misread():
    w = torch.zeros((3, 130, 272), dtype=torch.bfloat16)
    _refused(ops.fp8_quantize_weights, {"w": w}, {
        "fp32": {"w": w.float()}, "strided": {"w": _strided(w)}, "transposed": {"w": w.transpose(1, 2)}, "codes of another shape": {"codes": _f8(390, 272)},
        "codes of bytes": {"codes": torch.zeros((3, 130, 272), dtype=torch.uint8)}, "scales of 130 rows": {"scales": torch.zeros((3, 130, 3))},
        "scales of one matrix": {"scales": torch.zeros((2, 3))}, "scales over all rows": {"scales": torch.zeros((4, 3))}, "host tensors": {},
    })
    for bad, error in ((w[0, 0], ValueError), (w[None], ValueError), (None, TypeError)):
        with pytest.raises(error):
            ops.fp8_quantize_weights(bad)


def test_products_refuse_operands_they_would_misread():
    good = {"a": _f8(4, 272), "a_scales": torch.zeros((3, 4)), "w": _f8(260, 272), "w_scales": torch.zeros((3, 3))}
    _refused(ops.fp8_gemm, good, {
        "bytes": {"a": torch.zeros((4, 272), dtype=torch.uint8)}, "the other 8-bit type": {"a": torch.zeros((4, 272)).to(torch.float8_e5m2)}, "strided activations": {"a": _strided(_f8(4, 272))},
        "strided weights": {"w": _strided(_f8(260, 272))}, "weights of another K": {"w": _f8(260, 256)}, "scales a row of activations": {"a_scales": torch.zeros((4, 3))},
        "fp16 scales": {"a_scales": torch.zeros((3, 4), dtype=HALF)}, "scales of fewer blocks": {"w_scales": torch.zeros((2, 3))}, "scales of fewer k": {"w_scales": torch.zeros((3, 2))},
        "fp32 bias": {"bias": torch.zeros(260)}, "bias of another length": {"bias": torch.zeros(259, dtype=HALF)}, "residual of another shape": {"residual": torch.zeros((260, 4), dtype=HALF)},
        "two types": {"bias": torch.zeros(260, dtype=HALF), "residual": torch.zeros((4, 260), dtype=torch.bfloat16)},
        "another type than named": {"bias": torch.zeros(260, dtype=HALF), "dtype": torch.bfloat16}, "fp32 results": {"dtype": torch.float32}, "fp32 out": {"out": torch.zeros((4, 260))},
        "out of another shape": {"out": torch.zeros((4, 259), dtype=HALF)}, "another act": {"act": 2}, "odd rows of gate and up": {"act": 1, "w": _f8(259, 272), "w_scales": torch.zeros((4, 3))},
        "gate and up in one run of blocks": {"act": 1}, "out of both halves": {"act": 1, "w_scales": torch.zeros((4, 3)), "out": torch.zeros((4, 260), dtype=HALF)}, "host tensors": {},
    })
    for change, error in (({"a": _f8(4)}, ValueError), ({"w": _f8(272)}, ValueError), ({"a": None}, TypeError), ({"act": "1"}, TypeError), ({"dtype": "half"}, TypeError),
                          ({"variant": "tile_1x1"}, KeyError)):
        with pytest.raises(error):
            ops.fp8_gemm(**{**good, **change})


def test_the_grouped_product_refuses_operands_it_would_misread():
    good = {"a": _f8(4, 272), "a_scales": torch.zeros((3, 4)), "w": _f8(3, 260, 272), "w_scales": torch.zeros((3, 3, 3)), "offsets": torch.zeros(4, dtype=torch.int32)}
    _refused(ops.fp8_grouped_gemm, good, {
        "offsets without the end": {"offsets": torch.zeros(3, dtype=torch.int32)}, "int64 offsets": {"offsets": torch.zeros(4, dtype=torch.int64)},
        "strided offsets": {"offsets": torch.zeros(8, dtype=torch.int32)[::2]}, "weights of another K": {"w": _f8(3, 260, 256)}, "strided weights": {"w": _strided(_f8(3, 260, 272))},
        "scales of fewer experts": {"w_scales": torch.zeros((2, 3, 3))}, "scales of all rows": {"w_scales": torch.zeros((9, 3))}, "gate and up in one run of blocks": {"act": 1},
        "out of another shape": {"out": torch.zeros((4, 130), dtype=HALF)}, "fp32 results": {"dtype": torch.float32}, "another act": {"act": -1}, "host tensors": {},
    })
    for change, error in (({"w": _f8(260, 272)}, ValueError), ({"offsets": None}, TypeError)):
        with pytest.raises(error):
            ops.fp8_grouped_gemm(**{**good, **change})


# ---- at the C entry, with addresses that are never followed: every call below is refused, or finds no device


def _no_device():
    if torch.cuda.is_available():
        pytest.skip("made-up addresses: where there is a device, a call that is let through would run")


A, AS, W, WS, Y, B, R, X = ((i + 1) << 44 for i in range(8))


def _gemm(a=A, a_s=AS, w=W, w_s=WS, y=Y, type=1, m=4, n=64, k=256, bias=None, residual=None, act=0, variant=0):
    return _lib.kernels().nnf_fp8_gemm_variant(None, a, a_s, w, w_s, y, type, m, n, k, bias, residual, act, variant)


def _grouped(a=A, a_s=AS, w=W, w_s=WS, offsets=X, y=Y, type=0, experts=3, m=4, n=64, k=256, act=0, variant=0):
    return _lib.kernels().nnf_fp8_grouped_gemm_variant(None, a, a_s, w, w_s, offsets, y, type, experts, m, n, k, act, variant)


def test_products_refuse_bad_arguments_at_the_c_entry():
    _no_device()
    assert _gemm() == NO_DEVICE and _grouped() == NO_DEVICE
    for change in ({"a": None}, {"a_s": None}, {"w": None}, {"w_s": None}, {"y": None}, {"m": 0}, {"n": 0}, {"k": 0}, {"m": -1}, {"act": 2}, {"act": -1}, {"type": 2}, {"type": -1},
                   {"variant": -1}, {"variant": 11}, {"a": A + 8}, {"w": W + 1}, {"a_s": AS + 2}, {"w_s": WS + 1}, {"y": Y + 2}):
        assert _gemm(**change) == INVALID, change
        assert _grouped(**change) == INVALID, change
    for change in ({"bias": B + 2}, {"residual": R + 8}):
        assert _gemm(**change) == INVALID, change
    for change in ({"offsets": None}, {"experts": 0}, {"experts": -2}, {"offsets": X + 2}):
        assert _grouped(**change) == INVALID, change
    for change in ({"k": 40}, {"k": 8}, {"k": (1 << 22) + 16}, {"n": (1 << 29) + 1}, {"m": (1 << 30) + 1}, {"act": 1, "n": 1 << 16, "k": 1 << 15}):
        assert _gemm(**change) == UNSUPPORTED, change
        assert _grouped(**change) == UNSUPPORTED, change
    assert _gemm(act=1, bias=B) == UNSUPPORTED and _gemm(act=1, residual=R) == UNSUPPORTED
    for good in ({"a_s": AS + 4, "w_s": WS + 8}, {"k": 16, "m": 1, "n": 1}, {"n": 1 << 16, "k": 1 << 15}, {"m": 1 << 26}, {"act": 1, "k": 1 << 22, "n": 511}):
        assert _gemm(**good) == NO_DEVICE, good
        assert _grouped(**good) == NO_DEVICE, good
    for variant in range(1, 11):
        assert _gemm(variant=variant) == NO_DEVICE and _grouped(variant=variant, act=1) == NO_DEVICE
    # sizes whose tiles no grid holds, whichever kernel is asked for
    for variant in range(11):
        assert _gemm(m=1 << 28, n=1 << 12, k=32, variant=variant) == UNSUPPORTED
        assert _grouped(m=1 << 20, experts=1 << 20, n=4096, k=32, variant=variant) == UNSUPPORTED
    for experts in (2**31 - 1, 2**31 - 64, (1 << 30) + 1):
        assert _grouped(experts=experts, n=1, k=16) == UNSUPPORTED


def test_the_output_must_not_lie_on_an_operand():
    _no_device()
    row, scales, out = 256, 2 * 4 * 4, 4 * 64 * 2
    for change in ({"y": A}, {"y": A + 4 * row - 16}, {"a": Y + out - 16}, {"y": AS + scales - 16}, {"y": W + 64 * row - 16}, {"y": WS}):
        assert _gemm(**change) == INVALID, change
        assert _grouped(**change) == INVALID, change
    assert _gemm(y=A + 4 * row) == NO_DEVICE and _gemm(y=W + 64 * row) == NO_DEVICE
    assert _gemm(act=1, y=W + 128 * row - 16) == INVALID  # the up rows too
    assert _grouped(y=W + 3 * 64 * row - 16) == INVALID and _grouped(y=W + 3 * 64 * row) == NO_DEVICE
    assert _grouped(y=X) == INVALID and _gemm(bias=Y + 16) == INVALID
    assert _gemm(residual=Y) == NO_DEVICE and _gemm(residual=Y + 16) == INVALID  # the same place is fine, a shifted one is not


def test_quantising_refuses_bad_arguments_at_the_c_entry():
    _no_device()
    quantize, weights = _lib.kernels().nnf_fp8_quantize, _lib.kernels().nnf_fp8_quantize_weights
    good = (A, 0, None, W, WS, 4, 4, 272)
    assert quantize(None, *good) == NO_DEVICE and quantize(None, A, 1, X, W, WS, 9, 4, 272) == NO_DEVICE
    for args in ((None, 0, None, W, WS, 4, 4, 64), (A, 0, None, None, WS, 4, 4, 64), (A, 0, None, W, None, 4, 4, 64), (A, 2, None, W, WS, 4, 4, 64), (A, -1, None, W, WS, 4, 4, 64),
                 (A, 0, None, W, WS, 0, 0, 64), (A, 0, None, W, WS, 4, 4, 0), (A, 0, None, W, WS, 4, 5, 64), (A, 0, X, W, WS, 4, 0, 64), (A, 0, X, W, WS, -4, 4, 64),
                 (A + 8, 0, None, W, WS, 4, 4, 64), (A, 0, X + 2, W, WS, 4, 4, 64), (A, 0, None, W + 4, WS, 4, 4, 64), (A, 0, None, W, WS + 2, 4, 4, 64),
                 (A, 0, None, A, WS, 4, 4, 64), (A, 0, None, W, A + 508, 4, 4, 64), (A, 0, None, W, W, 4, 4, 64), (A, 0, X, X, WS, 4, 4, 64), (A, 0, X, W, X + 12, 4, 4, 64)):
        assert quantize(None, *args) == INVALID, args
    for rows, k in ((4, 40), (4, (1 << 22) + 16), ((1 << 24) + 1, 16), (1 << 24, 528)):
        assert quantize(None, A, 0, None, W, WS, rows, rows, k) == UNSUPPORTED
    assert quantize(None, A, 0, X, W, WS, 4, 2147483647, 1 << 12) == NO_DEVICE
    assert weights(None, A, 1, W, WS, 3, 130, 272) == NO_DEVICE
    for args in ((None, 0, W, WS, 1, 64, 64), (A, 0, None, WS, 1, 64, 64), (A, 0, W, None, 1, 64, 64), (A, 2, W, WS, 1, 64, 64), (A, 0, W, WS, 0, 64, 64), (A, 0, W, WS, 1, -1, 64),
                 (A, 0, W, WS, 1, 64, 0), (A + 2, 0, W, WS, 1, 64, 64), (A, 0, W + 8, WS, 1, 64, 64), (A, 0, W, WS + 2, 1, 64, 64), (A, 0, A, WS, 1, 64, 64), (A, 0, W, A, 1, 64, 64),
                 (A, 0, W, W + 4092, 1, 64, 64), (A, 0, A + 8176, WS, 1, 64, 64)):
        assert weights(None, *args) == INVALID, args
    assert weights(None, A, 0, W, WS, 1, 64, 40) == UNSUPPORTED
    assert weights(None, A, 0, W, WS, 1 << 23, 128, 128) == UNSUPPORTED and weights(None, A, 0, W, WS, (1 << 23) - 1, 128, 128) == NO_DEVICE
    assert weights(None, A, 0, W, WS, 2147483647, 2147483647, 16) == UNSUPPORTED


def test_the_c_entries_without_a_variant():
    _no_device()
    lib = _lib.kernels()
    assert lib.nnf_fp8_gemm(None, A, AS, W, WS, Y, 1, 4, 64, 256, B, R, 0) == NO_DEVICE
    assert lib.nnf_fp8_grouped_gemm(None, A, AS, W, WS, X, Y, 1, 3, 4, 64, 256, 1) == NO_DEVICE
    assert lib.nnf_fp8_gemm(None, A, AS, W, WS, Y, 1, 4, 64, 257, B, R, 0) == UNSUPPORTED
    assert lib.nnf_fp8_grouped_gemm(None, A, AS, W, WS, None, Y, 1, 3, 4, 64, 256, 1) == INVALID
