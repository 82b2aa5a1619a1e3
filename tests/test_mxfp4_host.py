"""The MXFP4 operators on the host side: the C++ unit tests of shape inference, emitters and the choice of a kernel
(tests/cpp/test_mxfp4.cpp), and the code generated for a mixture of experts, compiled here and run on the GPU."""
import os
import subprocess

import numpy as np
import pytest
import torch

from nnfusion_amd import datagen, ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BIN = os.path.join(ROOT, "nnfusion_amd", "bin")


def test_host_cpp_suite():
    proc = subprocess.run([os.path.join(BIN, "test_mxfp4")], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    lines = [l for l in proc.stdout.splitlines() if l.startswith(("PASS", "FAIL"))]
    assert proc.returncode == 0 and len(lines) >= 6 and all(l.startswith("PASS") for l in lines), proc.stdout


def test_generated_experts(tmp_path):
    """Four calls into the library, one per node, and the constants that the generator was asked for."""
    out = str(tmp_path / "rt") + "/"
    subprocess.run([os.path.join(BIN, "nnf_compile_example"), "mx_experts", out, "5", "64", "96"], check=True, timeout=60, stdout=subprocess.PIPE)
    text = open(out + "nnfusion_rt.cpp").read()
    assert text.count("NNF_HIP_CHECK(nnf_") == 4
    for call in ("nnf_mxfp4_quantize_f16(stream, input0, input1, output0, output1, 10, 5, 64)",
                 "nnf_mxfp4_grouped_gemm(stream, input0, input1, input2, input3, input4, output0, 4, 10, 96, 64, NNF_ACT_SILU_GATE, nullptr, 0)",
                 "nnf_mxfp4_quantize_f16(stream, input0, nullptr, output0, output1, 10, 10, 96)",
                 "nnf_mxfp4_grouped_gemm(stream, input0, input1, input2, input3, input4, output0, 4, 10, 64, 96, NNF_ACT_NONE, nullptr, 0)"):
        assert call in text, call
    sizes = sorted(os.path.getsize(out + "Constant/" + c) for c in os.listdir(out + "Constant"))
    assert sizes == sorted([4 * 192 * 32, 4 * 192 * 16, 4 * 64 * 48, 4 * 64 * 16])


@pytest.mark.gpu
def test_generated_experts_runtime(gpu):
    import test_codegen

    m, hidden, inter, experts = 37, 256, 416, 4
    x = datagen.normal_f16(0, datagen.S_ACT, (m, hidden))
    gen = torch.Generator()
    gen.manual_seed(1)
    to = torch.randint(0, experts - 1, (2 * m,), generator=gen)  # the last expert gets nothing
    order = torch.argsort(to, stable=True)
    index = (order // 2).int().numpy()
    offsets = np.concatenate([[0], np.cumsum(np.bincount(to.numpy(), minlength=experts))]).astype(np.int32)
    y = test_codegen._run_generated("mx_experts", [x, index, offsets], (2 * m, hidden), torch.float16, gpu)

    def matrix(codes, scales, n, k):  # the constants that the example was generated with
        c = datagen.uniform_u4_packed(0, codes, experts * n, k).reshape(experts, n, k // 2)
        s = datagen.uniform_i8(0, scales, (experts, n, ops.mxfp4_scale_bytes(k)), 118, 124).view(np.uint8)
        return torch.from_numpy(c).to(gpu), torch.from_numpy(s).to(gpu)

    # the same operators, called one by one, give the same bits (each is tested against 64-bit products elsewhere)
    groups = torch.from_numpy(offsets).to(gpu)
    a = ops.mxfp4_quantize(torch.from_numpy(x).to(gpu), torch.from_numpy(index).to(gpu))
    h = ops.mxfp4_grouped_gemm(*a, *matrix(datagen.S_WQ, datagen.S_MXS, 2 * inter, hidden), groups, act=1)
    want = ops.mxfp4_grouped_gemm(*ops.mxfp4_quantize(h), *matrix(datagen.S_WQ2, datagen.S_MXS2, hidden, inter), groups)
    assert torch.isfinite(want).all() and want.abs().max() > 0
    assert np.array_equal(y.view(np.int16), want.cpu().numpy().view(np.int16))
