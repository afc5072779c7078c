"""The library's host code against a HIP runtime that only keeps account of
device memory (tests/cpp/host_memory.cpp), so without a GPU."""

import pathlib
import subprocess

import pytest

BIN = pathlib.Path(__file__).resolve().parent / "cpp" / "host_memory"


def test_scratch_that_grows():
    if not BIN.exists():
        pytest.skip("tests/cpp/host_memory not built (run __graft_entry__.build())")
    r = subprocess.run([str(BIN)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "FAIL" not in r.stdout and "all are freed" in r.stdout, r.stdout + r.stderr
