"""The tile kernels ask for operands in LDS ahead of their use and wait for them by count, unseen by the compiler: along every path through the
machine code of the library built here, no instruction touches a register while a read into it may be under way.  (Scalar loads count in the same
counter and return when they like: a wait for `n` still leaves no more than n reads.)"""
import glob
import os
import re
import shutil
import subprocess

import pytest

LLVM = "/opt/rocm/llvm/bin"
LIBRARY = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nnfusion_amd", "lib", "libnnf_hip_kernels.so")


def registers(text):
    found = set()
    for first, last, one in re.findall(r"\bv\[(\d+):(\d+)\]|\bv(\d+)\b", text):
        found.update([int(one)] if one else range(int(first), int(last) + 1))
    return frozenset(found)


def conflicts(code):
    """code: (address, text, target of a branch or None) of each instruction -> what touches a register too early.  A state is the reads under way, oldest
    first, as sets of registers; LDS answers in order, so a wait for `n` leaves the last n."""
    at = {address: i for i, (address, _, _) in enumerate(code)}
    seen = [set() for _ in code]
    todo, bad = [(0, ())], []
    while todo:
        i, reads = todo.pop()
        while i < len(code) and reads not in seen[i]:
            seen[i].add(reads)
            _, text, target = code[i]
            op = text.split()[0]
            flying = frozenset().union(*reads)
            if flying & registers(text):
                bad.append(text)
            wait = re.search(r"lgkmcnt\((\d+)\)", text) if op == "s_waitcnt" else None
            if wait:
                reads = reads[max(len(reads) - int(wait.group(1)), 0):]
            elif op.startswith("ds_"):
                reads += (registers(text.split(",")[0]) if op.startswith("ds_read") else frozenset(),)
                assert len(reads) < 64, text
            while reads and not reads[0]:
                reads = reads[1:]
            if op == "s_endpgm":
                break
            if op == "s_branch":
                i = at[target]
                continue
            if op.startswith("s_cbranch"):
                todo.append((at[target], reads))
            i += 1
    return bad


def instructions(text):
    """llvm-objdump's lines -> conflicts()'s"""
    code = []
    for line in text.splitlines():
        m = re.match(r"\s+(\S.*?)\s*// ([0-9A-F]+):(?:.*<\S+\+0x([0-9a-f]+)>)?", line)
        if m:
            code.append((int(m.group(2), 16), m.group(1), int(m.group(3), 16) if m.group(3) else None))
    start = code[0][0]
    return [(address - start, text, target if text.startswith(("s_branch", "s_cbranch")) else None) for address, text, target in code]


def test_what_counts_as_too_early():
    def run(*lines):
        return len(conflicts([(4 * i, text, None if len(l) == 1 else l[1]) for i, l in enumerate(lines) for text in l[:1]]))

    read, use, end = ("ds_read_b128 v[4:7], v1",), ("v_add_f32 v0, v5, v5",), ("s_endpgm",)
    assert run(read, use, end) == 1
    assert run(read, ("s_waitcnt lgkmcnt(0)",), use, end) == 0
    assert run(read, ("ds_read_b32 v9, v1",), ("s_waitcnt lgkmcnt(1)",), use, end) == 0
    assert run(read, ("ds_write_b32 v1, v2",), ("s_waitcnt lgkmcnt(1)",), use, end) == 0
    assert run(("ds_read_b32 v9, v1",), read, ("s_waitcnt lgkmcnt(1)",), use, end) == 1
    assert run(read, ("v_mov_b32 v6, v0",), end) == 1 and run(read, ("v_mov_b32 v8, v0",), end) == 0
    assert run(read, ("s_waitcnt vmcnt(0)",), use, end) == 1
    assert run(read, ("s_load_dword s0, s[2:3], 0x0",), ("s_waitcnt lgkmcnt(1)",), use, end) == 1
    assert run(read, ("s_load_dword s0, s[2:3], 0x0",), ("s_waitcnt lgkmcnt(0)",), use, end) == 0
    # around a loop: the read of one turn, the use of the next
    assert run(("s_nop 0",), use, ("s_waitcnt lgkmcnt(0)",), read, ("s_cbranch_scc1 65532", 4), end) == 1
    assert run(("s_nop 0",), ("s_waitcnt lgkmcnt(0)",), use, read, ("s_cbranch_scc1 65532", 4), end) == 0


@pytest.mark.parametrize("kernel", ["fp8_tile_kernel", "mxfp4_tile_kernel", "w8a8_gemm_dl_kernel", "w4a16_gemm_sk_kernel"])
def test_nothing_touches_an_operand_on_its_way(tmp_path, kernel):
    if not os.path.exists(os.path.join(LLVM, "llvm-objdump")) or not os.path.exists(LIBRARY):
        pytest.skip("needs the built library and the ROCm LLVM tools")
    lib = shutil.copy(LIBRARY, tmp_path / "lib.so")
    subprocess.run([os.path.join(LLVM, "llvm-objdump"), "--offloading", str(lib)], cwd=tmp_path, check=True, stdout=subprocess.DEVNULL)
    checked = 0
    for code_object in glob.glob(str(tmp_path / "lib.so.*gfx950*")):
        if kernel.encode() not in open(code_object, "rb").read():
            continue
        text = subprocess.run([os.path.join(LLVM, "llvm-objdump"), "-d", code_object], check=True, capture_output=True, text=True).stdout
        for part in re.split(r"^[0-9a-f]+ <", text, flags=re.M)[1:]:
            name, _, body = part.partition(">:")
            if kernel in name:
                checked += 1
                assert not conflicts(instructions(body)), name
    assert checked >= 16
