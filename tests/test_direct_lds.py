"""The wait states that loads into LDS need and that the compiler does not keep for inline assembly, counted in the assembly of this framework's own code, without a GPU: one from a write of M0 to
the load that takes its place in LDS from there, five from a vector instruction's write of a scalar register to a memory instruction that reads it."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "turbofno_amd", "csrc")


def registers(operand):
    """scalar registers that an operand names"""
    m = re.fullmatch(r"s\[(\d+):(\d+)\]|s(\d+)", operand)
    if not m:
        return set()
    return {int(m[3])} if m[3] else set(range(int(m[1]), int(m[2]) + 1))


def instructions(source, tmp_path):
    out = str(tmp_path / "a.s")
    subprocess.run(["hipcc", "-O3", "-std=c++17", "--offload-arch=gfx950", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "-w", "--cuda-device-only", "-S", source, "-o", out], check=True,
                   stderr=subprocess.DEVNULL)
    for line in open(out):
        line = line.split(";")[0].strip()
        if line and line[0] != "." and not line.endswith(":"):
            name, _, operands = line.partition(" ")
            yield name, [o.strip() for o in operands.split(",")]


@pytest.mark.parametrize("source", [os.path.join(ROOT, "tests", "host", "direct_lds_check.hip"), os.path.join(CSRC, "mix_blocks.hip")])
def test_wait_states_ahead_of_loads_into_lds(source, tmp_path):
    code, loads = list(instructions(source, tmp_path)), 0
    for i, (name, operands) in enumerate(code):
        if not name.startswith("global_load_lds"):
            continue
        loads += 1
        base, states = registers(operands[1]), 0
        for before, what in reversed(code[max(0, i - 8):i]):
            writes = what[0] if what else ""
            assert states >= 1 or writes != "m0", (i, code[i - 3:i + 1])
            assert states >= 5 or not (before.startswith("v_") and registers(writes) & base), (i, code[i - 6:i + 1])
            states += int(what[0]) + 1 if before == "s_nop" else 1
    assert loads >= 5


def test_no_other_source_has_its_own():
    for name in os.listdir(CSRC):
        if name.endswith((".h", ".hip")) and name != "direct_lds.h":
            assert "load_lds" not in open(os.path.join(CSRC, name)).read(), name
