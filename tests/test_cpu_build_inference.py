"""The kernels of the forward pass in 8-bit integers on the CPU: whole translation units of the library, compiled with clang against
cpu_build/simt (workgroups as fibers), run through their own entry points under AddressSanitizer and UBSan, against 64-bit results.

Their inline assembly is replaced in a copy of the source, statement by statement: a load straight into LDS, its place, the waits and the
barriers by what they do (simt_inference.hpp), an empty one by nothing.  One that is not known here is an error."""
import json
import os
import re
import subprocess
import sys

import pytest

from verinf_amd.build import CSRC

HERE = os.path.dirname(os.path.abspath(__file__))
DIR = os.path.join(HERE, "cpu_build")
CLANG = os.environ.get("CLANGXX", "/opt/rocm/llvm/bin/clang++")
ASSEMBLY = [(r'asm volatile\("" : [^;]*\);', ";"),
            (r'asm volatile\("s_mov_b32 m0, %0" : : "s"\((\w+)\) : "memory"\);', r"simt::fetch_at(\1);"),
            (r'asm volatile\("s_nop 4\\n\\tglobal_load_lds_dwordx4 %0, %1\\n\\ts_add_u32 m0, m0, 0x1000" : : "v"\((\w+)\), "s"\(\w+\) : "memory", "scc"\);',
             r"simt::fetch(\1, (uint64_t)base);"),
            (r'asm volatile\("s_waitcnt vmcnt\(%0\) lgkmcnt\(0\)\\n\\ts_barrier" : : "n"\((\w+)\) : "memory"\);', r"simt::wait_for_loads_but(\1), __syncthreads();"),
            (r'asm volatile\("s_waitcnt lgkmcnt\(0\)\\n\\ts_barrier" : : : "memory"\);', "__syncthreads();"),
            (r"\(u32\)\(uintptr_t\)\(__attribute__\(\(address_space\(3\)\)\) char \*\)([\w.]+)", r"simt::lds_base(\1)")]


def _runtime():
    """clang's AddressSanitizer as a library to be loaded first; none: these tests cannot run"""
    if not os.path.exists(CLANG):
        return None
    so = subprocess.check_output([CLANG, "-print-file-name=libclang_rt.asan-x86_64.so"], text=True).strip()
    return so if os.path.isabs(so) and os.path.exists(so) else None


pytestmark = pytest.mark.skipif(not _runtime(), reason="no clang with AddressSanitizer")


def _build(unit, folder):
    for name in sorted(os.listdir(CSRC)):
        if name not in (unit + ".hip", "int8_gemm.hpp", "number_types.hpp", "common.hpp"):
            continue
        text = open(os.path.join(CSRC, name)).read()
        text = re.sub(r"#pragma unroll[^\n]*", "", text)        # a third of the compiler's time, and the loops are the same
        for pattern, meaning in ASSEMBLY:
            text = re.sub(pattern, meaning, text)
        code = re.sub(r"//[^\n]*", "", text)
        assert "asm" not in code and "address_space" not in code, name
        with open(os.path.join(folder, name), "w") as f:
            f.write(text.replace('"../../include/verinf_hip.h"', f'"{os.path.join(os.path.dirname(HERE), "include", "verinf_hip.h")}"'))
    so = os.path.join(folder, f"simt_{unit}.so")
    subprocess.check_call([CLANG, "-O2", "-g", "-std=c++17", "-fPIC", "-shared", "-rtlib=compiler-rt", "-ffp-contract=off", "-Wno-unknown-attributes", "-Wno-unused-value", "-Wno-psabi",
                           "-fsanitize=address,undefined", "-fno-sanitize=function,vptr", "-fno-sanitize-recover=undefined", "-shared-libasan", "-I", folder,
                           "-I", DIR, "-I", os.path.join(DIR, "simt"), "-o", so, os.path.join(DIR, f"simt_{unit}.cpp")])
    return so


@pytest.fixture(scope="module")
def built(tmp_path_factory):
    """One build per translation unit, made when a test first asks for it."""
    made, folder = {}, str(tmp_path_factory.mktemp("simt_inference"))
    return lambda unit: made[unit] if unit in made else made.setdefault(unit, _build(unit, folder))


def check(built, unit, what, **switches):
    env = dict(os.environ, LD_PRELOAD=_runtime(), ASAN_OPTIONS="detect_leaks=0,verify_asan_link_order=0", OPENBLAS_NUM_THREADS="1", **switches)
    res = subprocess.run([sys.executable, os.path.join(DIR, "simt_inference_checks.py"), what, built(unit)], stdout=subprocess.PIPE, stderr=subprocess.STDOUT,
                         text=True, env=env, timeout=600)
    assert res.returncode == 0 and res.stdout.strip().endswith("OK"), res.stdout[-4000:]


def test_log_probabilities_of_negative_zeros(built):
    check(built, "logprobs", "zeros")


def test_log_probabilities_of_few_allowed_entries(built):
    check(built, "logprobs", "few")


def test_log_probabilities_over_their_forms(built):
    check(built, "logprobs", "rows")


@pytest.mark.parametrize("how", ["direct", "staged", "copied", "sliced"])
def test_products_of_every_tile(built, how):
    check(built, "int8_gemm", how)


@pytest.mark.parametrize("how", ["direct", "copied", "sliced"])
def test_products_whose_loads_arrive_late(built, how):
    check(built, "int8_gemm", how, SIMT_LATE="1")


def test_products_of_few_rows(built):
    check(built, "int8_gemm", "few_rows")


def test_gated_products_that_overflow(built):
    check(built, "int8_gemm", "overflow")


def test_the_sizes_of_the_gpu_tests_take_every_tile(built):
    import test_gpu_inference as gpu
    check(built, "int8_gemm", "plans", SHAPES=json.dumps([gpu.LARGE, gpu.LARGE_GATED]))


def test_rows_to_8_bits(built):
    check(built, "quantize", "quantize")


def test_log_probabilities_of_logits_far_apart(built):
    check(built, "logprobs", "far")
