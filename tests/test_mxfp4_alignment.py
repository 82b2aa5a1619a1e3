"""Loads of the MXFP4 kernels for few rows promise the compiler no more alignment than their addresses have: a batch of steps begins at any word of
a row of scale bytes.  Read from the kernels' code as the front end hands it to the optimiser."""
import os
import re
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nnfusion_amd", "csrc")
HIPCC = "/opt/rocm/bin/hipcc"


def test_a_batch_s_scale_bytes_are_loaded_by_words(tmp_path):
    if not os.path.exists(HIPCC):
        pytest.skip("needs hipcc")
    out = str(tmp_path / "rows.ll")
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-std=c++17", "-O3", "-I" + os.path.join(CSRC, "../../include"), "--cuda-device-only", "-emit-llvm", "-S",
                    "-Xclang", "-disable-llvm-passes", "-o", out, os.path.join(CSRC, "kernels", "mxfp4_rows.hip")], check=True, timeout=300, stderr=subprocess.DEVNULL)
    bodies = re.findall(r"^define [^@\n]*@_ZZN\S*mxfp4_rows_kernel\S*\([^\n]*\{\n(.*?)^\}", open(out).read(), re.M | re.S)
    batches = [b for b in bodies if "llvm.amdgcn.mfma.scale" in b]
    by_words = [len(re.findall(r"load <4 x i32>, ptr %\d+, align 4\b", b)) for b in batches]
    assert len(batches) >= 15  # three kernels, batches of four steps and of one to four that end a range
    assert by_words == [2] * len(batches)  # of the weights and of the activations
