"""Runs the C++ test program of the 8-bit operators (tests/host/test_decx_f8_api.cpp, built by backup_1_amd/host/Makefile)."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BIN = os.path.join(ROOT, "tests", "build", "test_decx_f8_api")


def _run(mode):
    assert os.path.exists(BIN), "build it with `make -C backup_1_amd/host` (or __graft_entry__.build())"
    r = subprocess.run([BIN, mode], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    print(r.stdout)
    assert r.returncode == 0, r.stdout[-3000:]
    assert "0 failure(s)" in r.stdout


def test_f8_api_cpu_side():
    _run("cpu")


@pytest.mark.gpu
def test_f8_api_gpu_side():
    _run("gpu")
