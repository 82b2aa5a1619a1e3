"""Stores of more than eight bytes read their registers after they were issued: on these GPUs two instructions (or wait states) have to pass before a vector
instruction may write them.  The compiler sees to its own stores, not to those written as assembly: each of these has both wait states right behind it, and along
every path through the machine code of the library built here no such register is written sooner."""
import glob
import os
import re
import shutil
import subprocess

import pytest

LLVM = "/opt/rocm/llvm/bin"
LIBRARY = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nnfusion_amd", "lib", "libnnf_hip_kernels.so")
STATES = 2


def registers(text):
    found = set()
    for first, last, one in re.findall(r"\bv\[(\d+):(\d+)\]|\bv(\d+)\b", text):
        found.update([int(one)] if one else range(int(first), int(last) + 1))
    return found


def stored(text):
    """The registers whose contents a wide store writes to memory."""
    m = re.match(r"(?:global|flat|scratch)_store_dwordx[34]\s+\S+\s+(v\[\d+:\d+\])", text) or re.match(r"buffer_store_dwordx[34]\s+(v\[\d+:\d+\])", text)
    return registers(m.group(1)) if m else set()


def states(text):
    m = re.match(r"s_nop (\d+)", text)
    return int(m.group(1)) + 1 if m else 1


def too_early(code):
    """code: (text, index of a branch's target or None) -> the vector instructions that write a register less than STATES behind a store of it."""
    bad = []
    for i, (text, _) in enumerate(code):
        data = stored(text)
        todo = [(i + 1, 0)] if data else []
        while todo:
            at, passed = todo.pop()
            if at >= len(code) or passed >= STATES:
                continue
            line, target = code[at]
            op = line.split()[0]
            # (what a vector instruction writes comes first; of two results, or of both registers of a swap, a few more registers are looked at than need be)
            if op.startswith("v_") and data & registers(" ".join(line.split(",")[: 2 if "swap" in op else 1])):
                bad.append(f"{text} / {line}")
            if op == "s_endpgm":
                continue
            if target is not None:
                todo.append((target, passed + 1))
            if op != "s_branch":
                todo.append((at + 1, passed + states(line)))
    return bad


def instructions(text):
    """llvm-objdump's lines of one kernel -> too_early()'s"""
    lines = []
    for line in text.splitlines():
        m = re.match(r"\s+(\S.*?)\s*// ([0-9A-F]+):(?:.*<\S+\+0x([0-9a-f]+)>)?", line)
        if m:
            lines.append((int(m.group(2), 16), m.group(1), m.group(3)))
    at = {address - lines[0][0]: i for i, (address, _, _) in enumerate(lines)}
    return [(t, at[int(target, 16)] if t.startswith(("s_branch", "s_cbranch")) else None) for _, t, target in lines]


def test_what_counts_as_too_early():
    def run(*lines):
        return len(too_early([l if isinstance(l, tuple) else (l, None) for l in lines]))

    store, write, end = "global_store_dwordx4 v[8:9], v[0:3], off nt", "v_mov_b32_e32 v2, v9", "s_endpgm"
    assert run(store, write, end) == 1 and run(store, "s_nop 0", write, end) == 1 and run(store, "s_nop 1", write, end) == 0
    assert run(store, "s_mov_b32 s0, s1", "s_nop 0", write, end) == 0 and run(store, "v_mov_b32_e32 v8, v9", write, end) == 1
    assert run(store, "v_add_f32_e32 v4, v2, v3", "s_nop 0", write, end) == 0 and run(store, "v_cmp_eq_u32_e32 vcc, v2, v3", end) == 0
    assert run("global_store_dwordx4 v8, v[0:3], s[4:5]", write, end) == 1 and run("buffer_store_dwordx4 v[0:3], v8, s[4:7], 0 offen", write, end) == 1
    assert run("global_store_dwordx2 v[8:9], v[2:3], off", write, end) == 0 and run("global_load_dwordx4 v[0:3], v[8:9], off", write, end) == 0
    assert run(store, "v_mfma_f32_16x16x32_bf16 v[0:3], v[4:7], v[8:11], 0", end) == 1 and run(store, "v_permlane32_swap_b32_e32 v9, v2", end) == 1
    # the other end of a branch, and of a loop
    assert run(store, ("s_cbranch_scc1 1", 4), "s_nop 1", end, write, end) == 1 and run(store, ("s_branch 2", 3), write, "s_nop 0", end) == 0
    assert run(write, store, ("s_cbranch_scc1 65533", 0), end) == 1


def test_wide_stores_keep_their_registers(tmp_path):
    if not os.path.exists(os.path.join(LLVM, "llvm-objdump")) or not os.path.exists(LIBRARY):
        pytest.skip("needs the built library and the ROCm LLVM tools")
    lib = shutil.copy(LIBRARY, tmp_path / "lib.so")
    subprocess.run([os.path.join(LLVM, "llvm-objdump"), "--offloading", str(lib)], cwd=tmp_path, check=True, stdout=subprocess.DEVNULL)
    kernels, written = 0, 0
    for code_object in glob.glob(str(tmp_path / "lib.so.*gfx950*")):
        text = subprocess.run([os.path.join(LLVM, "llvm-objdump"), "-d", code_object], check=True, capture_output=True, text=True).stdout
        for part in re.split(r"^[0-9a-f]+ <", text, flags=re.M)[1:]:
            name, _, body = part.partition(">:")
            if "_store_dwordx" not in body:
                continue
            kernels += 1
            code = instructions(body)
            assert not too_early(code), name
            # stores of grouped products past the caches: the only ones that assembly in these kernels writes
            if "fp8_tile_kernel" in name:
                for (text, _), (behind, _) in zip(code, code[1:]):
                    if stored(text) and text.endswith(" off nt"):
                        written += 1
                        assert states(behind) >= STATES, (name, text, behind)
    assert kernels >= 100 and written >= 16
