"""What the compiler made of the kernels of routing, combining and block-scaled 8-bit floating point, read from the metadata of the library that was built
from them."""
import glob
import os
import re
import shutil
import subprocess

import pytest

LLVM = "/opt/rocm/llvm/bin"
LIBRARY = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nnfusion_amd", "lib", "libnnf_hip_kernels.so")


# Sums, operands of a step and of the next, and a lane's scores are held in registers; spilled ones would go through memory inside the loops.
def test_the_kernels_use_no_private_memory(tmp_path):
    if not os.path.exists(os.path.join(LLVM, "llvm-objdump")) or not os.path.exists(LIBRARY):
        pytest.skip("needs the built library and the ROCm LLVM tools")
    lib = shutil.copy(LIBRARY, tmp_path / "lib.so")
    subprocess.run([os.path.join(LLVM, "llvm-objdump"), "--offloading", str(lib)], cwd=tmp_path, check=True, stdout=subprocess.DEVNULL)
    seen, spilled = {"fp8": 0, "moe": 0}, []
    for code_object in glob.glob(str(tmp_path / "lib.so.*gfx950*")):
        notes = subprocess.run([os.path.join(LLVM, "llvm-readelf"), "--notes", code_object], check=True, capture_output=True, text=True).stdout
        for name, private in re.findall(r"\.name:\s+(_Z\S+)\n\s+\.private_segment_fixed_size:\s+(\d+)", notes):
            for kind in seen:
                if kind in name:
                    seen[kind] += 1
                    if int(private):
                        spilled.append((name, int(private)))
    assert seen["fp8"] >= 20 and seen["moe"] >= 10
    assert not spilled
