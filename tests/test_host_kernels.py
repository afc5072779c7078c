"""Which kernels a layer's operators take, against a HIP runtime that runs none
(tests/cpp/host_kernels.cpp), so without a GPU."""

import pathlib
import subprocess

import pytest

BIN = pathlib.Path(__file__).resolve().parent / "cpp" / "host_kernels"


def test_whole_pieces_only_where_rows_are_whole_and_the_kernels_that_the_tests_reach():
    if not BIN.exists():
        pytest.skip("tests/cpp/host_kernels not built (run __graft_entry__.build())")
    r = subprocess.run([str(BIN)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.startswith("0 failures"), r.stdout + r.stderr
