"""Attention over the cache and drafts on the CPU at the ends of numbers' ranges: cpu_build/simt_generation_edges.py over the builds of test_cpu_build_generation.py."""
import os
import subprocess
import sys

import pytest

from test_cpu_build_generation import _build
from test_cpu_build_inference import DIR, _runtime

pytestmark = pytest.mark.skipif(not _runtime(), reason="no clang with AddressSanitizer")


@pytest.fixture(scope="module")
def built(tmp_path_factory):
    made, folder = {}, str(tmp_path_factory.mktemp("simt_edges"))
    return lambda unit: made[unit] if unit in made else made.setdefault(unit, _build(unit, folder))


def check(built, unit, what):
    env = dict(os.environ, LD_PRELOAD=_runtime(), ASAN_OPTIONS="detect_leaks=0,verify_asan_link_order=0", OPENBLAS_NUM_THREADS="1")
    res = subprocess.run([sys.executable, os.path.join(DIR, "simt_generation_edges.py"), what, built(unit)], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, env=env, timeout=900)
    assert res.returncode == 0 and res.stdout.strip().endswith("OK"), res.stdout[-4000:]


def test_keys_far_above_those_before_them(built):
    check(built, "attention", "late_keys")


def test_weights_that_are_small_together(built):
    check(built, "attention", "small_weights_16")


def test_values_all_alike(built):
    check(built, "attention", "values_alike")


def test_scores_that_are_all_nothing(built):
    check(built, "attention", "small_scales")


def test_drafts_of_masked_tokens(built):
    check(built, "drafts", "masked_drafts")


def test_first_tokens_that_have_a_probability(built):
    check(built, "drafts", "first_tokens")


def test_logits_far_from_nothing(built):
    check(built, "drafts", "far_logits")


def test_few_tokens_left(built):
    check(built, "drafts", "few_tokens_left")


def test_numbers_next_to_the_border(built):
    check(built, "drafts", "next_to_the_border")
