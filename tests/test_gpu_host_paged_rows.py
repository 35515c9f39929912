"""Paged caches in 4 bits through the C++ host mirror on the GPU: runs
tests/cpp/test_paged_rows (rows written and read back, steps, commits)."""
import os
import subprocess

import pytest

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "test_paged_rows")


@pytest.mark.gpu
def test_cpp_paged_caches_in_4_bits():
    assert os.path.exists(BIN), "build the package first (tests/cpp/test_paged_rows missing)"
    r = subprocess.run([BIN], capture_output=True, text=True, timeout=110)
    print(r.stdout)
    print(r.stderr)
    assert r.returncode == 0, r.stderr
    assert "all" in r.stdout and "checks passed" in r.stdout
