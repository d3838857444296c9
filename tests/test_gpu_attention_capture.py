"""A paged attention call captured into a graph after eager calls of the same head_dim and cache type at other sizes: another
arrangement of its waves, and another host thread, need nothing from the runtime that a capture would not allow."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))

CHILD = """
import os, sys, threading
sys.path[:0] = [{here!r}, os.path.join(os.path.dirname({here!r}), "kvmem-qw3_amd")]
import numpy as np
from q8mi import hip
from test_gpu_paged_attention import Case
hip.set_device(0)
kind, dim, warm = sys.argv[1], int(sys.argv[2]), sys.argv[3]
# bounds that cut a call into tiles of one, two and four waves of rows
calls = dict(one=dict(lens=[40], rows=[1], far=True), two=dict(lens=[70], rows=[5], far=True), four=dict(lens=[90], rows=[1]))
cases = {{name: Case(heads=4, kv_heads=1, dim=dim, kind=kind, page=16, seed=i, **c) for i, (name, c) in enumerate(calls.items())}}
s = hip.Stream()
cases[warm].launch(s.handle)
s.synchronize()
cases[warm].check()


def replay(name):
    hip.set_device(0)
    c = cases[name]
    g = hip.Graph(s)
    with g:
        c.launch(s.handle)
    for _ in range(3):
        c.dout.fill(0x5a)
        hip.synchronize()
        g.launch()
        s.synchronize()
        c.check()
    print("replayed", name, flush=True)


for name in cases:
    replay(name) if name != "four" else None
t = threading.Thread(target=replay, args=("four",))   # a capture on a thread that has called nothing before
t.start()
t.join()
os._exit(0)
"""


@pytest.mark.parametrize("kind,dim,warm", [("bf16", 256, "one"), ("bf16", 256, "four"), ("f16", 128, "one"), ("e4m3", 256, "two"), ("bf16", 64, "one")])
def test_another_arrangement_is_captured(gpu, kind, dim, warm):
    """In a process of its own: what earlier tests have called must not matter."""
    r = subprocess.run([sys.executable, "-c", CHILD.format(here=HERE), kind, str(dim), warm], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout[-1000:] + r.stderr[-2000:]
    assert r.stdout.splitlines() == ["replayed one", "replayed two", "replayed four"], r.stdout + r.stderr[-2000:]
