"""Runs the C++ test program of results over inputs (tests/host/test_decx_f8_aliases.cpp, built by backup_1_amd/host/Makefile): on the
CPU over a device of host memory, which checks what each call reads and writes, and over the GPU."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PARTS = ("quantize", "gemm", "norm", "backward")


def _run(name, part):
    path = os.path.join(ROOT, "tests", "build", name)
    assert os.path.exists(path), "build it with `make -C backup_1_amd/host` (or __graft_entry__.build())"
    r = subprocess.run([path, part], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    print(r.stdout)
    assert r.returncode == 0, r.stdout[-3000:]
    assert part + ": 0 failure(s)" in r.stdout


@pytest.mark.parametrize("part", PARTS)
def test_results_over_inputs_on_the_cpu(part):
    _run("test_decx_f8_aliases", part)


@pytest.mark.gpu
@pytest.mark.parametrize("part", PARTS)
def test_results_over_inputs_on_the_gpu(part):
    _run("test_decx_f8_aliases_gpu", part)
