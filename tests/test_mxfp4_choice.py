"""The products named beside the constants of the MXFP4 kernels: at each, the choice of a kernel takes the one that it stands beside."""
import os
import re
import shutil
import subprocess

import pytest

PLAN = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nnfusion_amd", "csrc", "nnf_mxfp4_plan.h")

PROGRAM = """
#include "%s"
#include <stdio.h>
#include <stdlib.h>
int main(int argc, char** argv)
{
    for (int i = 1; i + 4 < argc; i += 5) // rows, columns of Y, K, gate, experts
        printf("%%d\\n", (int)nnf::mx::choose(atoi(argv[i]), atoi(argv[i + 1]), atoi(argv[i + 2]), atoi(argv[i + 3]) != 0, atoi(argv[i + 4]), 256));
}
"""


def test_the_products_beside_the_constants_take_those_kernels(tmp_path):
    if not shutil.which("g++"):
        pytest.skip("needs g++")
    text = open(PLAN).read()
    kernels = re.findall(r"^ +((?:ROWS|TILE)_\w+),", text, re.M)
    beside = re.findall(r"// ((?:ROWS|TILE)_\w+): (\d+) rows?(?: by|, (\d+) (?:uneven )?experts of) (\d+) x (\d+)(, SiLU-gate)?", text)
    assert len(kernels) == 15 and [b[0] for b in beside] == kernels
    arguments = []
    for _, rows, experts, weight_rows, k, gate in beside:
        arguments += [rows, str(int(weight_rows) // (2 if gate else 1)), k, "1" if gate else "0", experts or "0"]
    source, program = tmp_path / "choose.cpp", str(tmp_path / "choose")
    source.write_text(PROGRAM % PLAN)
    subprocess.run(["g++", "-O1", "-std=c++14", "-o", program, str(source)], check=True, timeout=60)
    out = subprocess.run([program] + arguments, check=True, capture_output=True, text=True, timeout=10).stdout.split()
    assert [kernels[int(c)] for c in out] == kernels
