"""Runs tests/cpp/backend_guards.cpp: what the host layer refuses of its own handles, and what one eager call with the
largest bounds prepares for captured ones."""
import os
import subprocess

import pytest

DRIVER = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "backend_guards")


@pytest.mark.gpu
def test_guards():
    assert os.path.exists(DRIVER), "the driver is not built (run __graft_entry__.build())"
    r = subprocess.run([DRIVER], capture_output=True, text=True, timeout=110)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
    assert [line for line in r.stdout.splitlines() if line.startswith("PASS")] == ["PASS frequencies", "PASS caches", "PASS captured"]
