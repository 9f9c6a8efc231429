"""Runs the C++ test program of where results and inputs lie to each other (tests/host/test_operands.cpp)."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BIN = os.path.join(ROOT, "tests", "build", "test_operands")


def test_operands_against_their_bytes():
    assert os.path.exists(BIN), "build it with `make -C backup_1_amd/host` (or __graft_entry__.build())"
    r = subprocess.run([BIN], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    print(r.stdout)
    assert r.returncode == 0 and "0 failure(s)" in r.stdout, r.stdout[-3000:]
