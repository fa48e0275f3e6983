"""The C++ host mirror's calls for packed tokens and caches in pages, through their own test program (tests/cpp/paged_mirror_test.cpp)."""
import os
import subprocess

import pytest

CPP = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp")


def run(what):
    subprocess.check_call(["make", "-s", "-C", CPP, "paged_mirror_test"])
    r = subprocess.run([os.path.join(CPP, "paged_mirror_test"), what], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stdout + r.stderr


def test_cpp_refusals_need_no_gpu():
    run("errors")


def test_cpp_host_positions_are_checked():
    run("rows")


@pytest.mark.gpu
def test_cpp_prompts_and_steps():
    run("gpu")


@pytest.mark.gpu
def test_cpp_a_prefix_on_the_device_is_read_once():
    run("prefix")
