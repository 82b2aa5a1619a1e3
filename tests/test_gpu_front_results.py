"""The results that the calls allocate are torch's like any other: modes see them made, and where torch is asked for deterministic memory they are filled."""
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from nnfusion_amd import ops

pytestmark = pytest.mark.gpu


class Allocations(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.made = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        out = func(*args, **(kwargs or {}))
        if func is torch.ops.aten.empty.memory_format:
            self.made.append((tuple(out.shape), out.dtype))
        return out


@pytest.fixture
def deterministic():
    was, filled = torch.are_deterministic_algorithms_enabled(), torch.utils.deterministic.fill_uninitialized_memory
    torch.use_deterministic_algorithms(True)
    torch.utils.deterministic.fill_uninitialized_memory = True
    yield
    torch.use_deterministic_algorithms(was)
    torch.utils.deterministic.fill_uninitialized_memory = filled


def _operands(gpu):
    x = torch.randn((48, 256), generator=torch.Generator().manual_seed(1)).half().to(gpu)
    w = torch.randn((4 * 64, 256), generator=torch.Generator().manual_seed(2)).half().to(gpu)
    return x, w


def _calls(gpu):
    """name, the call, what it allocates"""
    x, w = _operands(gpu)
    m_a, m_w, f_a = ops.mxfp4_quantize(x), ops.mxfp4_quantize(w), ops.fp8_quantize(x)
    f_w = ops.fp8_quantize_weights(w.view(4, 64, 256))
    offsets = torch.tensor([0, 10, 10, 30, 40], dtype=torch.int32, device=gpu)
    routed = ops.moe_route(x[:, :8].contiguous(), 2)
    half, u8, f8, f32, i32 = torch.float16, torch.uint8, torch.float8_e4m3fn, torch.float32, torch.int32
    stride = m_a[1].shape[1]
    return [
        ("mxfp4_quantize", lambda: ops.mxfp4_quantize(x), [((48, 128), u8), ((48, stride), u8)]),
        ("mxfp4_dequantize", lambda: ops.mxfp4_dequantize(*m_a), [((48, 256), half)]),
        ("mxfp4_gemm", lambda: ops.mxfp4_gemm(*m_a, *m_w), [((48, 256), half)]),
        ("mxfp4_grouped_gemm", lambda: ops.mxfp4_grouped_gemm(*m_a, m_w[0].view(4, 64, -1), m_w[1].view(4, 64, -1), offsets), [((48, 64), half)]),
        ("moe_route", lambda: ops.moe_route(x[:, :8].contiguous(), 2, out=(None,) * 5), [((48, 2), f32), ((48, 2), i32), ((96,), i32), ((9,), i32), ((48, 2), i32)]),
        ("moe_combine", lambda: ops.moe_combine(x, routed[0], routed[4]), [((48, 256), half)]),
        ("fp8_quantize", lambda: ops.fp8_quantize(x), [((48, 256), f8), ((2, 48), f32)]),
        ("fp8_quantize_weights", lambda: ops.fp8_quantize_weights(w), [((256, 256), f8), ((2, 2), f32)]),
        ("fp8_gemm", lambda: ops.fp8_gemm(*f_a, f_w[0][0], f_w[1][0]), [((48, 64), half)]),
        ("fp8_grouped_gemm", lambda: ops.fp8_grouped_gemm(*f_a, *f_w, offsets), [((48, 64), half)]),
    ]


def test_modes_see_the_results_made(gpu):
    for name, call, want in _calls(gpu):
        call()
        with Allocations() as mode:
            call()
        for result in want:
            assert result in mode.made, (name, result, mode.made)


def test_deterministic_memory_is_filled(gpu, deterministic):
    """Rows that belong to no group: NaN, as torch fills what nobody writes."""
    for name, call, _ in _calls(gpu):
        result = call()
        if "grouped" in name:
            assert bool(torch.isnan(result[40:]).all()) and not bool(torch.isnan(result[:40]).any()), name


def test_results_made_under_inference_mode(gpu):
    with torch.inference_mode():
        for name, call, _ in _calls(gpu):
            results = call()
            assert all(t.is_inference() for t in (results if isinstance(results, tuple) else (results,))), name
