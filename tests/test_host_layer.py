"""The refusals, launches and scratch of a layer's operators against a HIP
runtime that runs no kernel (tests/cpp/host_layer.cpp), so without a GPU."""

import pathlib
import subprocess

import pytest

BIN = pathlib.Path(__file__).resolve().parent / "cpp" / "host_layer"


def test_refusals_and_launches():
    if not BIN.exists():
        pytest.skip("tests/cpp/host_layer not built (run __graft_entry__.build())")
    r = subprocess.run([str(BIN)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "FAIL" not in r.stdout and "0 failures" in r.stdout, r.stdout + r.stderr
