"""The loads straight into LDS of attention over the cache, in the listing of its kernels: their place is written to M0 in front of each and nothing else uses M0, and five
wait states lie between a vector instruction's write of the scalar address and the load."""
import os
import re
import shutil
import subprocess

import pytest

from test_cpu_build_int8_waits import HIPCC, WAIT_STATES, registers, wait_states_before
from verinf_amd.build import CSRC, FLAGS


@pytest.mark.skipif(not shutil.which(HIPCC), reason="no hipcc")
def test_loads_to_lds_wait_for_their_address_and_place(tmp_path):
    listing = str(tmp_path / "attention.s")
    flags = [f for f in FLAGS if f != "-fPIC"]
    subprocess.check_call([HIPCC] + flags + ["--cuda-device-only", "-S", "-o", listing, os.path.join(CSRC, "attention.hip")])
    kernels = re.findall(r"^(\S*k_attend\S*):[^\n]*\n(.*?)\.Lfunc_end", open(listing).read(), re.S | re.M)
    seen = {"global_load_lds_dwordx4": 0, "global_load_lds_dword": 0}
    assert len(kernels) == 18                                          # 3 kinds of cache, 3 widths of heads, 2 forms
    for name, body in kernels:
        instructions = [s for s in (line.split(";")[0].strip() for line in body.splitlines()) if s and s[0] not in "._" and not s.endswith(":")]
        for i, s in enumerate(instructions):
            op = s.split()[0]
            if op in seen:
                seen[op] += 1
                assert instructions[i - 1].startswith("s_nop") and re.match(r"s_mov_b32 m0, (s\d+|vcc_lo|vcc_hi)$", instructions[i - 2]), (name, instructions[i - 3:i + 1])
                if op == "global_load_lds_dwordx4":
                    base = registers(s.rsplit(", ", 1)[1])
                    assert base and wait_states_before(instructions, i, base) >= WAIT_STATES, (name, instructions[i - 6:i + 1])
            else:
                assert not re.search(r"\bm0\b", s) or re.match(r"s_mov_b32 m0, (s\d+|vcc_lo|vcc_hi)$", s), (name, s)
            assert not s.startswith("scratch_"), (name, s)             # waits that count loads have none of the compiler's between
    assert seen["global_load_lds_dwordx4"] > 200 and seen["global_load_lds_dword"] >= 12
