"""The device's status word when the very first call of a process is captured into a graph: it is not the graph's, so what an
eager call reports is still there after a replay."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PROGRAM = """
import torch
from verified_metal_kernels_b200 import _lib
from verified_metal_kernels_b200.kernels import pages_b200, prompt_b200
dev = torch.device("cuda", 0)
ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
junk = torch.full((1 << 25,), -1, dtype=torch.int32, device=dev)        # memory that comes back is not zero
del junk
torch.cuda.empty_cache()
q, k = torch.randn(40, 8, 128, device=dev).half(), torch.randn(40, 2, 128, device=dev).half()
cu, bad = ints([0, 40]), ints([0, 400])
table, lens, refs, keep, wrong = ints([[-1, -1]]), ints([0]), ints([0, 0]), ints([0]), ints([-1])
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    %s
assert _lib.read_status(dev) == 0                                       # before any replay
g.replay()
%s
g.replay()
torch.cuda.synchronize()
assert _lib.read_status(dev) == 2, "the replay took back what was reported"
assert _lib.read_status(dev) == 0
del g
%s
torch.cuda.synchronize()
assert _lib.read_status(dev) == 2
print("fine")
"""
FIRST = {"prompt": ("out = prompt_b200.kernel(q, k, k, cu)", "prompt_b200.kernel(q, k, k, bad)"),
         "pages": ("pages_b200.free(table, lens, refs, keep, 64)", "pages_b200.free(table, lens, refs, wrong, 64)")}


@pytest.mark.parametrize("first", FIRST)
def test_first_call_of_a_process_captured(first):
    good, report = FIRST[first]
    r = subprocess.run([sys.executable, "-c", PROGRAM % (good, report, report)], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "fine" in r.stdout, r.stdout + r.stderr
