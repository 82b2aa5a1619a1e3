"""Routing, combining and the block-scaled 8-bit operators on the host side: the C++ unit tests of shape inference, emitters and the choice of a kernel
(tests/cpp/test_fp8_moe.cpp), and the code generated for a mixture of experts, compiled here and run on the GPU."""
import os
import subprocess

import numpy as np
import pytest
import torch

from nnfusion_amd import datagen, ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BIN = os.path.join(ROOT, "nnfusion_amd", "bin")


def test_host_cpp_suite():
    proc = subprocess.run([os.path.join(BIN, "test_fp8_moe")], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    lines = [l for l in proc.stdout.splitlines() if l.startswith(("PASS", "FAIL"))]
    assert proc.returncode == 0 and len(lines) >= 7 and all(l.startswith("PASS") for l in lines), proc.stdout


def test_generated_experts(tmp_path):
    """Six calls into the library, one per node, and the constants that the generator was asked for."""
    out = str(tmp_path / "rt") + "/"
    subprocess.run([os.path.join(BIN, "nnf_compile_example"), "fp8_experts", out, "5", "64", "96"], check=True, timeout=60, stdout=subprocess.PIPE)
    text = open(out + "nnfusion_rt.cpp").read()
    assert text.count("NNF_HIP_CHECK(nnf_") == 6
    for call in ("const nnf_moe_routing routing = {3, NNF_MOE_SIGMOID, 4, 2, 2, 1, (float)2.5",
                 "nnf_moe_route(stream, input0, NNF_TYPE_F32, input1, nullptr, &routing, output0, output1, output2, output3, output4, 5, 8, nullptr, 0)",
                 "nnf_fp8_quantize(stream, input0, NNF_TYPE_F16, input1, output0, output1, 15, 5, 64)",
                 "nnf_fp8_grouped_gemm(stream, input0, input1, input2, input3, input4, output0, NNF_TYPE_F16, 8, 15, 96, 64, NNF_ACT_SILU_GATE)",
                 "nnf_fp8_quantize(stream, input0, NNF_TYPE_F16, nullptr, output0, output1, 15, 15, 96)",
                 "nnf_fp8_grouped_gemm(stream, input0, input1, input2, input3, input4, output0, NNF_TYPE_F16, 8, 15, 64, 96, NNF_ACT_NONE)",
                 "nnf_moe_combine(stream, input0, input1, input2, input3, output0, NNF_TYPE_F16, 5, 15, 3, 64)"):
        assert call in text, call
    sizes = sorted(os.path.getsize(out + "Constant/" + c) for c in os.listdir(out + "Constant"))
    assert sizes == sorted([8 * 192 * 64, 8 * 2 * 4, 8 * 64 * 96, 8 * 4])


@pytest.mark.gpu
def test_generated_experts_runtime(gpu):
    import test_codegen

    m, hidden, inter, experts = 37, 272, 400, 8
    x = datagen.normal_f16(0, datagen.S_ACT, (m, hidden))
    gen = torch.Generator()
    gen.manual_seed(1)
    logits, bias = torch.randn((m, experts), generator=gen), 0.1 * torch.randn((experts,), generator=gen)
    y = test_codegen._run_generated("fp8_experts", [x, logits.numpy(), bias.numpy()], (m, hidden), torch.float16, gpu)

    def matrix(codes, scales, parts, n, k):  # the constants that the example was generated with
        v = datagen.uniform_i8(0, codes, (experts, parts * n, k), -111, 111).astype(np.int32)
        c = np.where(v < 0, 0x80 | -v, v).astype(np.uint8)
        s = datagen.uniform_f32(0, scales, (experts, parts * ((n + 127) // 128), (k + 127) // 128), 0.0005, 0.002)
        return torch.from_numpy(c).view(torch.float8_e4m3fn).to(gpu), torch.from_numpy(s).to(gpu)

    # the same operators, called one by one, give the same bits (each is tested against 64 bits elsewhere)
    x = torch.from_numpy(x).to(gpu)
    weights, _, rows, offsets, positions = ops.moe_route(logits.to(gpu), 3, score="sigmoid", bias=bias.to(gpu), groups=4, top_groups=2, group_top=2, scale=2.5)
    h = ops.fp8_grouped_gemm(*ops.fp8_quantize(x, rows=rows), *matrix(datagen.S_WQ, datagen.S_MXS, 2, inter, hidden), offsets, act=1)
    down = ops.fp8_grouped_gemm(*ops.fp8_quantize(h), *matrix(datagen.S_WQ2, datagen.S_MXS2, 1, hidden, inter), offsets)
    want = ops.moe_combine(down, weights, positions, residual=x)
    assert torch.isfinite(want).all() and (want - x).abs().max() > 0
    assert np.array_equal(y.view(np.int16), want.cpu().numpy().view(np.int16))
