"""The C++ host mirror's calls for caches that are kept small, through their own test program (tests/cpp/cache_mirror_test.cpp)."""
import os
import subprocess

import pytest

CPP = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp")


def run(what):
    subprocess.check_call(["make", "-s", "-C", CPP, "cache_mirror_test"])
    r = subprocess.run([os.path.join(CPP, "cache_mirror_test"), what], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stdout + r.stderr


def test_cpp_refusals_need_no_gpu():
    run("errors")


@pytest.mark.gpu
def test_cpp_loop_of_append_attention_and_eviction():
    run("gpu")
