"""The kernels of the cache, of attention over it and of drafts on the CPU: whole translation units of the library, compiled with clang against cpu_build/simt, run
through their own entry points under AddressSanitizer and UBSan, against 64-bit results.

Their inline assembly is replaced in a copy of the source, statement by statement, by what it does (simt_generation.hpp).  One that is not known here is an error."""
import os
import re
import subprocess
import sys

import pytest

from test_cpu_build_inference import CLANG, DIR, HERE, _runtime
from verinf_amd.build import CSRC

ASSEMBLY = [(r'asm volatile\(""(?: : [^;]*)?\);', ";"),
            (r'asm volatile\("s_mov_b32 m0, %0\\n\\ts_nop 4\\n\\tglobal_load_lds_dwordx4 %1, %2" : : "s"\((\w+)\), "v"\((\w+)\), "s"\((\w+)\) : "memory"\);',
             r"simt::fetch16(\1, \2, (uint64_t)base);"),
            (r'asm volatile\("s_mov_b32 m0, %0\\n\\ts_nop 0\\n\\tglobal_load_lds_dword %1, off" : : "s"\((\w+)\), "v"\((\w+)\) : "memory"\);', r"simt::fetch4(\1, \2);"),
            (r'asm volatile\("s_waitcnt vmcnt\(%0\) lgkmcnt\(0\)" : : "n"\((\w+)\) : "memory"\);', r"simt::arrived_but(\1);"),
            (r'asm volatile\("s_waitcnt lgkmcnt\(0\)" : : : "memory"\);', ";"),
            (r'asm volatile\("s_barrier" : : : "memory"\);', "__syncthreads();"),
            (r"\(u32\)\(uintptr_t\)\(__attribute__\(\(address_space\(3\)\)\) char \*\)([\w.]+)", r"simt::lds_base(\1)"),
            (r"__attribute__\(\(address_space\([34]\)\)\) ?", "")]

pytestmark = pytest.mark.skipif(not _runtime(), reason="no clang with AddressSanitizer")


def _build(unit, folder, planted=None):
    for name in (unit + ".hip", "cache.hpp", "number_types.hpp", "common.hpp"):
        text = re.sub(r"#pragma unroll[^\n]*", "", open(os.path.join(CSRC, name)).read())
        if planted and name == unit + ".hip":
            assert planted[0] in text
            text = text.replace(*planted)
        for pattern, meaning in ASSEMBLY:
            text = re.sub(pattern, meaning, text)
        assert "asm" not in re.sub(r"//[^\n]*", "", text), name
        with open(os.path.join(folder, name), "w") as f:
            f.write(text.replace('"../../include/verinf_hip.h"', f'"{os.path.join(os.path.dirname(HERE), "include", "verinf_hip.h")}"'))
    so = os.path.join(folder, f"simt_{unit}.so")
    subprocess.check_call([CLANG, "-O1", "-g", "-std=c++17", "-fPIC", "-shared", "-rtlib=compiler-rt", "-ffp-contract=off", "-Wno-unknown-attributes", "-Wno-unused-value", "-Wno-psabi",
                           "-fsanitize=address,undefined", "-fno-sanitize=function,vptr", "-fno-sanitize-recover=undefined", "-shared-libasan", "-I", folder,
                           "-I", DIR, "-I", os.path.join(DIR, "simt"), "-o", so, os.path.join(DIR, f"simt_{unit}.cpp")])
    return so


@pytest.fixture(scope="module")
def built(tmp_path_factory):
    """One build per translation unit, made when a test first asks for it."""
    made, folder = {}, str(tmp_path_factory.mktemp("simt_generation"))
    return lambda unit: made[unit] if unit in made else made.setdefault(unit, _build(unit, folder))


def run(so, what, **switches):
    env = dict(os.environ, LD_PRELOAD=_runtime(), ASAN_OPTIONS="detect_leaks=0,verify_asan_link_order=0", OPENBLAS_NUM_THREADS="1", **switches)
    return subprocess.run([sys.executable, os.path.join(DIR, "simt_generation_checks.py"), what, so], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True,
                          env=env, timeout=900)


def check(built, unit, what, **switches):
    res = run(built(unit), what, **switches)
    assert res.returncode == 0 and res.stdout.strip().endswith("OK"), res.stdout[-4000:]


def test_heads_are_turned(built):
    check(built, "positions", "rotate")


def test_tokens_are_appended(built):
    check(built, "positions", "append")


def test_attention_of_both_forms(built):
    check(built, "attention", "attend")


def test_attention_whose_loads_arrive_late(built):
    check(built, "attention", "late", SIMT_LATE="1")


def test_drafts_are_verified(built):
    check(built, "drafts", "drafts")


def test_accepted_entries_move(built):
    check(built, "drafts", "keep")


# a wait for fewer loads than there are, in each of the two loops, and loads asked for before the last readers are done
@pytest.mark.parametrize("mistake", [("if (now_whole) arrive<LOADS_OF_HALF>();", "if (now_whole) arrive<LOADS_OF_HALF + 1>();"),
                                     ("if (next_whole) arrive<LOADS_OF_HALF>();", "if (next_whole) arrive<LOADS_OF_HALF + 1>();"),
                                     ("if (next_all) arrive<LOADS_OF_HALF>();", "if (next_all) arrive<2 * LOADS_OF_HALF>();")])
def test_a_wait_for_fewer_loads_is_found(tmp_path, mistake):
    assert run(_build("attention", str(tmp_path), mistake), "late", SIMT_LATE="1").returncode != 0


def test_loads_over_what_is_still_read_are_found(tmp_path):
    mistake = ("fetch(0, place_of(0, own), stage_key(it + 2), behind, behind_all);", "fetch(0, place_of(0, other), stage_key(it + 2), behind, behind_all);")
    assert run(_build("attention", str(tmp_path), mistake), "attend").returncode != 0
