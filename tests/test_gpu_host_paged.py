"""Paged caches through the C++ host mirror (HipPool, HipSequence over it,
xwfes_amd/host/) on the GPU: runs tests/cpp/test_paged_host, which compares
steps, commits and truncations with a contiguous cache's and exhausts a pool."""
import os
import subprocess

import pytest

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "test_paged_host")


@pytest.mark.gpu
def test_cpp_paged_caches():
    assert os.path.exists(BIN), "build the package first (tests/cpp/test_paged_host missing)"
    r = subprocess.run([BIN], capture_output=True, text=True, timeout=110)
    print(r.stdout)
    print(r.stderr)
    assert r.returncode == 0, r.stderr
    assert "all" in r.stdout and "checks passed" in r.stdout
