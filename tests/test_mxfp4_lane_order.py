"""Lanes of the MXFP4 tile kernels hand each other results through LDS: the order of their writes and reads has to be stated, or the
compiler may move accesses that are apart lane by lane.  Read from the kernels' code as the front end hands it to the optimiser."""
import os
import re
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nnfusion_amd", "csrc")
HIPCC = "/opt/rocm/bin/hipcc"


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """name -> the calls and fences of a kernel's own body, in their order"""
    if not os.path.exists(HIPCC):
        pytest.skip("needs hipcc")
    out = str(tmp_path_factory.mktemp("ir") / "tile.ll")
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-std=c++17", "-O3", "-I" + os.path.join(CSRC, "../../include"), "--cuda-device-only", "-emit-llvm", "-S",
                    "-Xclang", "-disable-llvm-passes", "-o", out, os.path.join(CSRC, "kernels", "mxfp4_tile.hip")], check=True, timeout=300, stderr=subprocess.DEVNULL)
    text = open(out).read()
    return text, dict(re.findall(r"^define [^@\n]*amdgpu_kernel [^@\n]*@(\S*mxfp4_tile_kernel\w+)\([^\n]*\{\n(.*?)^\}", text, re.M | re.S))


def _parameters(name):
    """WM, WN, WK, FM, FN, .. of the tile"""
    return [int(v) for v in re.findall(r"Li(\d+)E", name[name.index("4TileI"):])]


def test_lanes_wait_for_each_other_s_results(kernels):
    """A wavefront's block of results: written, ordered, read; ordered again before the next block of rows is written over it.  Where the
    wavefronts of a workgroup have ranges of K each, they meet at a barrier; else the lanes of one wavefront do."""
    text, bodies = kernels
    assert len(bodies) == 26  # thirteen tiles, with SiLU-gate and without
    helper = re.findall(r"^define [^\n]*@(\S*lanes_meet\S*)\([^\n]*\{\n(.*?)^\}", text, re.M | re.S)
    ordered = {}
    for name, body in helper:
        fences = re.findall(r'fence syncscope\("wavefront"\) (\w+)', body)
        ordered[name] = "s_barrier" in body or (fences == ["release", "acquire"] and "llvm.amdgcn.wave.barrier" in body)
    for name, body in bodies.items():
        at = [m.group(1) for m in re.finditer(r"call [^\n]*@(\S*lanes_meet\S*)\(", body)]
        assert len(at) == 2 and all(ordered[h] for h in at), (name, _parameters(name), at)


def test_no_barrier_of_the_workgroup_inside_the_blocks_of_one_wavefront(kernels):
    """The wavefronts of a tile over all of K have blocks of their own: ordering them costs no instruction."""
    text, bodies = kernels
    for name in bodies:
        if _parameters(name)[2] == 1:
            for h in re.findall(r"call [^\n]*@(\S*lanes_meet\S*)\(", bodies[name]):
                body = re.search(r"^define [^\n]*@" + re.escape(h) + r"\([^\n]*\{\n(.*?)^\}", text, re.M | re.S).group(1)
                assert "asm" not in body, name
