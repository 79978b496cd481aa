"""The C++ API of the appends that rotate and of caches held in 4 bits
(engine::hip::rope_append, q4_rope_append, q4_gather, q4_decode, q4_prefill and
PagedKVCache's 4-bit format), used together from C++ by tests/cpp/test_q4.  The binary
is built by tests/cpp/Makefile; it is built here only when missing."""
import os
import subprocess

import pytest

CPP = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp")
BIN = os.path.join(CPP, "test_q4")


def _run(mode, timeout):
    if not os.path.exists(BIN):
        subprocess.run(["make", "-s", "test_q4"], cwd=CPP, check=True)
    r = subprocess.run([BIN, mode], capture_output=True, text=True, timeout=timeout)
    assert r.returncode == 0 and " 0 failures" in r.stdout, r.stdout[-4000:] + r.stderr[-1000:]


def test_cpp_q4_refusals():
    _run("--cpu", 60)


@pytest.mark.gpu
def test_cpp_q4_served():
    _run("--gpu", 110)
