"""The gfx950 code of libbkv.so: loads straight into LDS keep the wait states that the hardware does not keep for
them. They are written in inline assembly, inside which the compiler looks for no hazards. (No counterpart in the
reference. No GPU: the built library is disassembled.)

 - M0, the LDS address, written by a scalar instruction: one wait state before the load that uses it.
 - An address pair in scalar registers written by a vector instruction (v_readfirstlane): five."""
import os
import re
import shutil
import subprocess

import pytest

from bonsai_vk_amd._lib import LIB_PATH

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
LOAD = re.compile(r"(global|scratch|buffer)_load_lds_|buffer_load_\w+ .*\blds\b")


def kernels(tmp):
    """Instructions of each code object, as (mnemonic, operands)."""
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    lib = shutil.copy(LIB_PATH, tmp)               # (the code objects are written beside the file)
    subprocess.run([OBJDUMP, "--offloading", lib], check=True, capture_output=True, cwd=tmp)
    objects = sorted(f for f in os.listdir(tmp) if f.endswith("gfx950"))
    assert objects, "no gfx950 code in the library"
    for f in objects:
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "--no-leading-addr", os.path.join(tmp, f)], check=True,
                              capture_output=True, text=True).stdout
        lines = [x.split("//")[0].strip() for x in text.splitlines()]
        yield f, [(x.split(None, 1)[0], x.split(None, 1)[1] if " " in x else "") for x in lines if x and not x.endswith(":")]


def wait_states(op, args):
    return int(args, 0) + 1 if op == "s_nop" else 1


def writes(op, args, regs):
    """Whether the instruction's destination is one of the scalar registers."""
    dst = args.split(",")[0].strip()
    m = re.fullmatch(r"s(?:(\d+)|\[(\d+):(\d+)\])", dst)
    if not m:
        return dst in regs
    lo = int(m[1] or m[2])
    return any(f"s{i}" in regs for i in range(lo, int(m[1] or m[3]) + 1))


def too_close(code, at, regs, need, writer):
    waits = 0
    for op, args in reversed(code[max(0, at - need):at]):
        if waits >= need:
            return False
        if writer(op) and writes(op, args, regs):
            return True
        waits += wait_states(op, args)
    return False


def faults(code):
    for at, (op, args) in enumerate(code):
        if not LOAD.match(f"{op} {args}"):
            continue
        if too_close(code, at, {"m0"}, 1, lambda o: o.startswith("s_")):
            yield at, "M0"
        m = re.search(r"\bs\[(\d+):(\d+)\]", args)
        if m and too_close(code, at, {f"s{i}" for i in range(int(m[1]), int(m[2]) + 1)}, 5, lambda o: o.startswith("v_")):
            yield at, "address"


def test_the_check_finds_what_it_looks_for():
    load, based = ("global_load_lds_dwordx4", "v[2:3], off"), ("global_load_lds_dwordx4", "v2, s[4:5]")
    m0, nop = ("s_mov_b32", "m0, s7"), ("s_nop", "0")
    assert [x for _, x in faults([m0, load])] == ["M0"] and not list(faults([m0, nop, load]))
    lane = ("v_readfirstlane_b32", "s5, v9")
    assert [x for _, x in faults([lane, m0, nop, ("s_nop", "1"), based])] == ["address"]
    assert not list(faults([lane, m0, nop, ("s_nop", "2"), based])) and not list(faults([("s_add_u32", "s4, s4, s9"), based]))


def test_loads_into_lds_keep_their_wait_states(tmp_path):
    loads = 0
    for name, code in kernels(str(tmp_path)):
        loads += sum(bool(LOAD.match(f"{op} {args}")) for op, args in code)
        bad = list(faults(code))
        assert not bad, (name, len(bad), [(what, code[at - 3:at + 1]) for at, what in bad[:3]])
    assert loads > 100, "the library's loads into LDS are not recognised any more"
