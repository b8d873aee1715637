"""The built library's loads to LDS, which are written in assembly: wait states that the compiler does not keep for them are there.

On gfx950 a memory instruction needs five after a vector instruction's write of a scalar register that it reads, and a load to LDS
one after m0's."""

import os
import re
import struct
import subprocess

import pytest

import npeff_ref_amd as d
from npeff_ref_amd import binding

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def device_objects():
    """The library's gfx950 code objects that hold tiles."""
    data = open(binding.LIB_PATH, "rb").read()
    at = data.find(MAGIC)
    while at >= 0:
        (n,) = struct.unpack_from("<Q", data, at + len(MAGIC))
        entry = at + len(MAGIC) + 8
        for _ in range(n):
            offset, size, length = struct.unpack_from("<QQQ", data, entry)
            if b"gfx950" in data[entry + 24 : entry + 24 + length]:
                code = data[at + offset : at + offset + size]
                if b"k_tiles" in code:
                    yield code
            entry += 24 + length
        at = data.find(MAGIC, at + len(MAGIC))


def registers(operands):
    found = {int(m) for m in re.findall(r"\bs(\d+)\b", operands)}
    for lo, hi in re.findall(r"\bs\[(\d+):(\d+)\]", operands):
        found |= set(range(int(lo), int(hi) + 1))
    return found


def faults(lines):
    """(loads to LDS, those that come too early), in the order in which the code lies."""
    before, loads, early = [], 0, []
    for line in lines:
        line = line.split("//")[0].strip()
        if not line or line.endswith(":"):
            continue
        name, _, operands = line.partition(" ")
        if name.startswith("buffer_load") and operands.endswith("lds"):
            loads += 1
            reads, states = registers(operands), 0
            for other, its in reversed(before[-8:]):
                if states < 5 and other.startswith("v_") and registers(its.split(",")[0]) & reads:
                    early.append((other, its, line))
                if states < 1 and its.startswith("m0"):
                    early.append((other, its, line))
                states += int(its, 0) + 1 if other == "s_nop" else 1
        before = before[-8:] + [(name, operands)]
    return loads, early


def test_wait_states_are_told_apart():
    load = "buffer_load_dwordx4 v5, s[4:7], 0 offen lds"
    good = ["v_readfirstlane_b32 s5, v1", "s_mov_b32 m0, s9", "s_nop 3", load]
    assert faults(good) == (1, [])
    assert len(faults(["v_readfirstlane_b32 s5, v1", "s_mov_b32 m0, s9", "s_nop 2", load])[1]) == 1
    assert len(faults(["s_mov_b32 m0, s9", load])[1]) == 1
    assert faults(["v_readfirstlane_b32 s8, v1", "s_mov_b32 m0, s9", "s_nop 0", load]) == (1, [])


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no disassembler")
def test_loads_of_the_library(tmp_path):
    assert d.size_of_split(1, 1, 0) == 1
    loads = 0
    for i, code in enumerate(device_objects()):
        path = tmp_path / f"{i}.o"
        path.write_bytes(code)
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "--mcpu=gfx950", str(path)], capture_output=True, text=True, check=True)
        n, early = faults(text.stdout.splitlines())
        assert not early, early[:5]
        loads += n
    assert loads > 100
