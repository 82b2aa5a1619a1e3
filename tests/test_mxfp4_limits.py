"""Sizes at the ends of what the MXFP4 calls take: refused before a device is asked for."""
import ctypes

from nnfusion_amd import _lib

UNSUPPORTED = -2

# addresses that are never followed, far enough apart for the largest operands
A, AS, W, WS, Y, X = (ctypes.c_void_p((i + 1) << 44) for i in range(6))


def _gemm(m, n, k=32, act=0, variant=0):
    return _lib.kernels().nnf_mxfp4_gemm_variant(None, A, AS, W, WS, Y, m, n, k, None, None, act, variant, None, 0)


def _grouped(experts, m=4, n=1, k=32, act=0):
    return _lib.kernels().nnf_mxfp4_grouped_gemm(None, A, AS, W, WS, X, Y, experts, m, n, k, act, None, 0)


def test_groups_whose_numbers_a_turn_of_64_would_carry_past_an_int():
    """The search for a tile looks at 64 groups a turn: the number of the first one behind the last group has to be an int too."""
    for experts in (2**31 - 1, 2**31 - 64, (1 << 30) + 1):
        assert _grouped(experts) == UNSUPPORTED
        assert _grouped(experts, act=1) == UNSUPPORTED


def test_products_that_no_grid_holds():
    """Refused whichever kernel is asked for, and where the library chooses."""
    for variant in range(16):
        assert _gemm(1 << 28, 1 << 12, variant=variant) == UNSUPPORTED
    assert _grouped(1 << 20, m=1 << 20, n=4096) == UNSUPPORTED  # (each expert may need a block of rows of its own)
    assert _grouped(1 << 23, m=1 << 23, n=1 << 16, act=1) == UNSUPPORTED
