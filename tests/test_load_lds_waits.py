"""The built kernels' direct loads into LDS, from their own disassembly (no GPU needed): the wait states that the
hardware wants before them, which the compiler does not add in inline assembly."""
import os
import re
import subprocess
import tempfile

import pytest

from helexa_amd import moe as hx

pytest.importorskip("msgpack")
from test_mxfp4_code import code_objects  # noqa: E402

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
pytestmark = pytest.mark.skipif(not os.path.exists(hx.LIB_PATH) or not os.path.exists(OBJDUMP), reason="no library or no disassembler")


def instructions(elf):
    with tempfile.NamedTemporaryFile(suffix=".co") as f:
        f.write(elf)
        f.flush()
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", f.name], capture_output=True, text=True, check=True).stdout
    for line in text.splitlines():
        yield line.split("//")[0].strip()


def states(before):
    """(instruction, wait states between it and the load) from the load backwards"""
    w = 0
    for ins in reversed(before):
        yield ins, w
        nop = re.match(r"s_nop (\d+)", ins)
        w += int(nop[1]) + 1 if nop else 1


def test_waits_before_direct_loads():
    """one state after a write of M0, five after a VALU instruction that writes the scalar address"""
    with open(hx.LIB_PATH, "rb") as f:
        lib = f.read()
    loads = 0
    for elf in code_objects(lib):
        before = []
        for ins in instructions(elf):
            if not ins or ins.endswith(":"):
                before = []
                continue
            if "load_lds" in ins:
                loads += 1
                address = re.search(r", s\[(\d+):(\d+)\]", ins)
                regs = range(int(address[1]), int(address[2]) + 1) if address else ()
                for other, w in states(before):
                    assert w >= 1 or not re.match(r"s_\w+ m0,", other), (other, ins)
                    lane = re.match(r"v_read(?:first)?lane_b32 s(\d+)", other)
                    assert w >= 5 or not lane or int(lane[1]) not in regs, (other, ins)
            before = (before + [ins])[-8:]
    assert loads > 100
