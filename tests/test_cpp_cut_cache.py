"""PagedKVCache::rope_append into caches that were cut, from C++ (tests/cpp/test_cut_cache,
built by tests/cpp/Makefile; it is built here only when missing)."""
import os
import subprocess

import pytest

CPP = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp")
BIN = os.path.join(CPP, "test_cut_cache")


@pytest.mark.gpu
def test_cpp_cut_cache():
    if not os.path.exists(BIN):
        subprocess.run(["make", "-s", "test_cut_cache"], cwd=CPP, check=True)
    r = subprocess.run([BIN, "--gpu"], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and " 0 failures" in r.stdout, r.stdout[-4000:] + r.stderr[-1000:]
