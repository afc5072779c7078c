"""The operators that answer with codes through include/aq_mi355x.hpp:
tests/cpp/code_step runs norm, 4-bit product and sampling in a chain and checks
each against its definition in doubles."""

import pathlib
import subprocess

import pytest

BIN = pathlib.Path(__file__).resolve().parent / "cpp" / "code_step"


def _run():
    if not BIN.exists():
        pytest.skip("tests/cpp/code_step not built (run __graft_entry__.build())")
    return subprocess.run([str(BIN)], capture_output=True, text=True, timeout=100)


def test_without_gpu_reports_it():
    import torch

    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    r = _run()
    assert r.returncode == 77 and "no GPU" in r.stdout, r.stdout + r.stderr


@pytest.mark.gpu
def test_chain_on_gpu():
    r = _run()
    print(r.stdout, flush=True)
    assert r.returncode == 0 and "FAIL" not in r.stdout, r.stdout + r.stderr
