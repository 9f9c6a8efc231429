"""Runs the C++ test program of the library's runtime record (tests/host/test_runtime_record.cpp)."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BIN = os.path.join(ROOT, "tests", "build", "test_runtime_record")


def test_raster_groups_asked_for():
    assert os.path.exists(BIN), "build it with `make -C backup_1_amd/host` (or __graft_entry__.build())"
    r = subprocess.run([BIN], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=60)
    assert r.returncode == 0 and "0 failure(s)" in r.stdout, r.stdout
