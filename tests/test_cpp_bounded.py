"""The C++ API of the caches of bounded length (engine::hip::window_decode,
window_prefill, weighted_decode, prompt_weights, evict_plan, evict_apply and
PagedKVCache::shrink), used together from C++ by tests/cpp/test_bounded.  The
binary is built by tests/cpp/Makefile; it is built here only when missing."""
import os
import subprocess

import pytest

CPP = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp")
BIN = os.path.join(CPP, "test_bounded")


def _run(mode, timeout):
    if not os.path.exists(BIN):
        subprocess.run(["make", "-s", "test_bounded"], cwd=CPP, check=True)
    r = subprocess.run([BIN, mode], capture_output=True, text=True, timeout=timeout)
    assert r.returncode == 0 and " 0 failures" in r.stdout, r.stdout[-4000:] + r.stderr[-1000:]


def test_cpp_bounded_refusals():
    _run("--cpu", 60)


@pytest.mark.gpu
def test_cpp_bounded_served():
    _run("--gpu", 110)
