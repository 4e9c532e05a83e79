"""gfx950 wants five wait states between a vector instruction's write of a scalar register and a vector memory instruction that reads it.
The compiler keeps them, but not in front of an instruction inside an asm block, as the 8-bit products' loads straight into LDS are: with
fewer the load takes the register's old value for its address.  The listing of the kernels is looked through for them, and for uses of M0,
which holds the place in LDS between those loads."""
import os
import re
import shutil
import subprocess

import pytest

from verinf_amd.build import CSRC, FLAGS

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
WAIT_STATES = 5


def registers(operand):
    m = re.match(r"s\[(\d+):(\d+)\]$", operand) or re.match(r"s(\d+)()$", operand)
    return set(range(int(m.group(1)), int(m.group(2) or m.group(1)) + 1)) if m else set()


def wait_states_before(instructions, at, base):
    """How many lie between the last vector instruction that writes one of the registers and the instruction `at`."""
    waited = 0
    for s in reversed(instructions[:at]):
        if waited >= WAIT_STATES:
            break
        op, _, operands = s.partition(" ")
        if op == "s_nop":
            waited += int(operands) + 1
            continue
        if op.startswith("v_") and registers(operands.split(",")[0].strip()) & base:
            break
        waited += 1
    return waited


def test_the_check_finds_a_load_too_near():
    near = ["v_readfirstlane_b32 s7, v1", "s_nop 0", "global_load_lds_dwordx4 v2, s[6:7]"]
    assert wait_states_before(near, 2, {6, 7}) == 1
    assert wait_states_before(["v_readfirstlane_b32 s7, v1", "s_nop 4"], 2, {6, 7}) == WAIT_STATES
    assert wait_states_before(["v_readfirstlane_b32 s9, v1"] + ["s_add_u32 s6, s6, 64"] * 5, 6, {6, 7}) == WAIT_STATES


@pytest.mark.skipif(not shutil.which(HIPCC), reason="no hipcc")
def test_loads_to_lds_wait_for_their_scalar_base(tmp_path):
    listing = str(tmp_path / "int8.s")
    flags = [f for f in FLAGS if f != "-fPIC"]
    subprocess.check_call([HIPCC] + flags + ["--cuda-device-only", "-S", "-o", listing, os.path.join(CSRC, "int8_gemm.hip")])
    kernels = re.findall(r"^(\S*k_tile\S*):[^\n]*\n(.*?)\.Lfunc_end", open(listing).read(), re.S | re.M)
    seen = 0
    for name, body in kernels:
        instructions = [s for s in (line.split(";")[0].strip() for line in body.splitlines()) if s and s[0] not in "._" and not s.endswith(":")]
        for i, s in enumerate(instructions):
            if s.startswith("global_load_lds"):
                seen += 1
                base = registers(s.rsplit(", ", 1)[1])
                assert base, (name, s)
                assert wait_states_before(instructions, i, base) >= WAIT_STATES, (name, instructions[i - 6:i + 1])
                assert instructions[i - 1].startswith("s_nop"), (name, instructions[i - 1])             # and one after a write of M0
            elif re.search(r"\bm0\b", s):
                assert re.match(r"s_mov_b32 m0, s\d+$|s_add_u32 m0, m0, 0x1000$", s), (name, s)
    assert seen > 200
