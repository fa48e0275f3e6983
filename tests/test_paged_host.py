"""The host code of packed tokens and caches in pages on the CPU (tests/cpp/paged_host_test.cpp): what its entries hand to their kernels."""
import os
import subprocess

import pytest

CPP = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp")


@pytest.mark.parametrize("name", [
    "a_call_without_kv_heads_reads_no_table",
    "a_call_without_kv_heads_has_no_last_row",
    "a_prefix_is_read_once_where_that_is_shorter",
])
def test_host_code(name):
    subprocess.check_call(["make", "-s", "-C", CPP, "paged_host_test"])
    r = subprocess.run([os.path.join(CPP, "paged_host_test"), name], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.strip().endswith("ok")
