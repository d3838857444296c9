"""Runs the C++ decode loop (tests/cpp/backend_decode.cpp): cache append, paged attention and sampling together, through the
host layer, between the projections and behind the LM head."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DRIVER = os.path.join(ROOT, "tests", "cpp", "backend_decode")


@pytest.mark.gpu
def test_decode_loop():
    assert os.path.exists(DRIVER), "the decode driver is not built (run __graft_entry__.build())"
    r = subprocess.run([DRIVER], capture_output=True, text=True, timeout=110)
    print(r.stdout)
    print(r.stderr)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
    assert [line.split(":")[0] for line in r.stdout.splitlines() if line.startswith("PASS")] == ["PASS attention", "PASS tokens", "PASS graph", "PASS refusals"]


def test_host_library_exports_the_operators():
    """No GPU needed."""
    lib = os.path.join(ROOT, "kvmem-qw3_amd", "host", "libq8mi_host.so")
    out = subprocess.run(["nm", "-DC", "--defined-only", lib], capture_output=True, text=True, check=True).stdout
    for method in ("qk_norm_rope_append(", "paged_attention(", "sample_rows(", "kv_cache(", "rope_frequencies(", "tensor_i32(", "tensor_i64("):
        assert f"qw3::HipQ8Backend::{method}" in out, method
