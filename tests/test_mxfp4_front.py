"""What the MXFP4 calls refuse, on host tensors and at the C entry points: nothing here reaches a kernel."""
import ctypes

import pytest
import torch

import mxfp4_reference as ref
from nnfusion_amd import _lib, ops

INVALID, UNSUPPORTED = -1, -2


def _packed(rows, k, *lead):
    return torch.zeros((*lead, rows, k // 2), dtype=torch.uint8), torch.zeros((*lead, rows, ref.scale_bytes(k)), dtype=torch.uint8)


def _strided(t):
    return torch.cat([t, t], dim=-1)[..., ::2]


@pytest.mark.parametrize("k", [32, 64, 480, 512, 544, 4096, 11008])
def test_scale_bytes(k):
    assert ops.mxfp4_scale_bytes(k) == ref.scale_bytes(k)


def test_quantising_refuses_what_it_would_misread():
    x = torch.zeros((4, 96), dtype=torch.float16)
    rows = torch.zeros(4, dtype=torch.int32)
    codes, scales = _packed(4, 96)
    for what, args in {
        "bf16": (x.bfloat16(),), "fp32": (x.float(),), "strided": (_strided(x),), "int64 rows": (x, rows.long()), "rows of two axes": (x, rows[None]),
        "strided rows": (x, torch.zeros(8, dtype=torch.int32)[::2]), "codes of fewer rows": (x, None, codes[:3], scales),
        "codes of another K": (x, None, codes[:, :32].contiguous(), scales), "signed codes": (x, None, codes.to(torch.int8), scales),
        "unpadded scales": (x, None, codes, scales[:, :3].contiguous()), "buffers of x's rows, not of the index": (x, rows[:2], codes, scales),
        "host tensors": (x,),
    }.items():
        with pytest.raises(AssertionError):
            ops.mxfp4_quantize(*args)
            pytest.fail(what)
    for args, error in (((x[0],), ValueError), ((None,), TypeError), ((x.numpy(),), TypeError), ((x, [0, 1]), TypeError)):
        with pytest.raises(error):
            ops.mxfp4_quantize(*args)


def test_reading_back_refuses_what_it_would_misread():
    codes, scales = _packed(4, 96)
    for args in ((codes.to(torch.int8), scales), (_strided(codes), scales), (codes, scales[:3].contiguous()), (codes, scales[:, :3].contiguous()),
                 (codes, scales, torch.zeros((4, 96))), (codes, scales, torch.zeros((4, 48), dtype=torch.float16)), (codes, scales)):
        with pytest.raises(AssertionError):
            ops.mxfp4_dequantize(*args)


def test_products_refuse_operands_they_would_misread():
    a, a_s = _packed(4, 96)
    w, w_s = _packed(32, 96)
    good = {"a": a, "a_scales": a_s, "w": w, "w_scales": w_s}
    half = torch.float16
    bad = {
        "signed codes": {"a": a.to(torch.int8)}, "strided activations": {"a": _strided(a)}, "strided weights": {"w": _strided(w)},
        "weights of another K": {"w": w[:, :32].contiguous()}, "scales of fewer rows": {"a_scales": a_s[:3].contiguous()},
        "unpadded scales": {"w_scales": w_s[:, :3].contiguous()}, "fp32 bias": {"bias": torch.zeros(32)}, "bias of another length": {"bias": torch.zeros(31, dtype=half)},
        "residual of another shape": {"residual": torch.zeros((4, 31), dtype=half)}, "strided residual": {"residual": torch.zeros((4, 64), dtype=half)[:, ::2]},
        "fp32 out": {"out": torch.zeros((4, 32))}, "out of another shape": {"out": torch.zeros((4, 31), dtype=half)}, "another act": {"act": 2},
        "odd rows of gate and up": {"act": 1, "w": w[:31].contiguous(), "w_scales": w_s[:31].contiguous()},
        "out of both halves": {"act": 1, "out": torch.zeros((4, 32), dtype=half)}, "fp32 workspace": {"workspace": torch.zeros(64)}, "host tensors": {},
    }
    for what, change in bad.items():
        with pytest.raises(AssertionError):
            ops.mxfp4_gemm(**{**good, **change})
            pytest.fail(what)
    for change, error in (({"a": a[0]}, ValueError), ({"w": w[0]}, ValueError), ({"a": None}, TypeError), ({"act": "1"}, TypeError), ({"act": 1 << 40}, OverflowError)):
        with pytest.raises(error):
            ops.mxfp4_gemm(**{**good, **change})


def test_the_grouped_product_refuses_operands_it_would_misread():
    a, a_s = _packed(4, 96)
    w, w_s = _packed(32, 96, 3)
    good = {"a": a, "a_scales": a_s, "w": w, "w_scales": w_s, "offsets": torch.zeros(4, dtype=torch.int32)}
    bad = {
        "offsets without the end": {"offsets": torch.zeros(3, dtype=torch.int32)}, "int64 offsets": {"offsets": torch.zeros(4, dtype=torch.int64)},
        "strided offsets": {"offsets": torch.zeros(8, dtype=torch.int32)[::2]}, "weights of another K": {"w": w[..., :32].contiguous()},
        "scales of fewer experts": {"w_scales": w_s[:2].contiguous()}, "out of another shape": {"out": torch.zeros((4, 64), dtype=torch.float16)},
        "another act": {"act": -1}, "host tensors": {},
    }
    for what, change in bad.items():
        with pytest.raises(AssertionError):
            ops.mxfp4_grouped_gemm(**{**good, **change})
            pytest.fail(what)
    for change, error in (({"w": w[0]}, ValueError), ({"offsets": None}, TypeError)):
        with pytest.raises(error):
            ops.mxfp4_grouped_gemm(**{**good, **change})


# addresses that are never followed: every call below is refused before a device is asked for
A, AS, W, WS, Y, B, R, X = (ctypes.c_void_p((i + 1) << 32) for i in range(8))


def _gemm(a=A, a_s=AS, w=W, w_s=WS, y=Y, m=4, n=64, k=256, bias=None, residual=None, act=0):
    return _lib.kernels().nnf_mxfp4_gemm(None, a, a_s, w, w_s, y, m, n, k, bias, residual, act, None, 0)


def _grouped(a=A, a_s=AS, w=W, w_s=WS, offsets=X, y=Y, experts=3, m=4, n=64, k=256, act=0):
    return _lib.kernels().nnf_mxfp4_grouped_gemm(None, a, a_s, w, w_s, offsets, y, experts, m, n, k, act, None, 0)


def _off(p, by):
    return ctypes.c_void_p(p.value + by)


def test_entry_points_refuse_bad_arguments():
    for change in ({"a": None}, {"a_s": None}, {"w": None}, {"w_s": None}, {"y": None}, {"m": 0}, {"n": 0}, {"k": 0}, {"m": -1}, {"act": 2}, {"act": -1}, {"a": _off(A, 8)},
                   {"w_s": _off(WS, 4)}, {"y": _off(Y, 2)}):
        assert _gemm(**change) == INVALID, change
        assert _grouped(**change) == INVALID, change
    for change in ({"bias": _off(B, 2)}, {"residual": _off(R, 8)}):
        assert _gemm(**change) == INVALID, change
    for change in ({"offsets": None}, {"experts": 0}, {"experts": -2}, {"offsets": _off(X, 4)}):
        assert _grouped(**change) == INVALID, change
    for change in ({"k": 48}, {"k": 33}, {"k": (1 << 22) + 32}, {"k": 8}):
        assert _gemm(**change) == UNSUPPORTED, change
        assert _grouped(**change) == UNSUPPORTED, change
    assert _gemm(act=1, bias=B) == UNSUPPORTED and _gemm(act=1, residual=R) == UNSUPPORTED
    assert _gemm(n=(1 << 29) + 1) == UNSUPPORTED


def test_the_output_must_not_lie_on_an_operand():
    row, scale, out = 128, 16, 4 * 64 * 2
    for change in ({"y": A}, {"y": _off(A, 4 * row - 16)}, {"a": _off(Y, out - 16)}, {"y": _off(AS, 4 * scale - 16)}, {"y": _off(W, 64 * row - 16)}, {"y": _off(WS, 64 * scale - 16)}):
        assert _gemm(**change) == INVALID, change
        assert _grouped(**change) == INVALID, change
    assert _gemm(act=1, y=_off(W, 128 * row - 16)) == INVALID  # the up rows too
    assert _grouped(y=_off(W, 3 * 64 * row - 16)) == INVALID
    assert _grouped(y=X) == INVALID
    assert _gemm(bias=_off(Y, 16)) == INVALID
    assert _gemm(residual=_off(Y, 16)) == INVALID  # the same place is fine, a shifted one is not


def test_conversions_refuse_bad_arguments():
    quantize, dequantize = _lib.kernels().nnf_mxfp4_quantize_f16, _lib.kernels().nnf_mxfp4_dequantize_f16
    for args in ((None, None, W, WS, 4, 4, 64), (A, None, None, WS, 4, 4, 64), (A, None, W, None, 4, 4, 64), (A, None, W, WS, 0, 0, 64), (A, None, W, WS, 4, 4, 0),
                 (A, None, W, WS, 4, 5, 64), (A, X, W, WS, 4, 0, 64), (_off(A, 8), None, W, WS, 4, 4, 64), (A, _off(X, 4), W, WS, 4, 4, 64), (A, None, _off(W, 4), WS, 4, 4, 64),
                 (A, None, A, WS, 4, 4, 64), (A, None, W, A, 4, 4, 64), (A, None, W, W, 4, 4, 64), (A, X, X, WS, 4, 4, 64)):
        assert quantize(None, *args) == INVALID, args
    assert quantize(None, A, None, W, WS, 4, 4, 40) == UNSUPPORTED
    assert quantize(None, A, X, W, WS, 1 << 28, 4, 32) == UNSUPPORTED  # more threads than a grid has
    for args in ((None, WS, Y, 4, 64), (W, None, Y, 4, 64), (W, WS, None, 4, 64), (W, WS, Y, 0, 64), (W, WS, Y, 4, -32), (W, WS, _off(Y, 8), 4, 64), (W, WS, W, 4, 64), (W, WS, WS, 4, 64)):
        assert dequantize(None, *args) == INVALID, args
    assert dequantize(None, W, WS, Y, 4, 24) == UNSUPPORTED
    assert dequantize(None, W, WS, Y, 1 << 27, 1024) == UNSUPPORTED
