"""The dense operators' first call of a process inside a stream capture: nothing they set up on first use may
be something that a capture does not allow."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CODE = """
import sys
import torch
from nano_ktrans_b200 import DenseMoeLayer, gated_linear, linear
m = int(sys.argv[1])
r = lambda *s: torch.randn(*s, device="cuda").to(torch.bfloat16) * 0.1
x, w, g, u, d, wr = r(m, 256), r(264, 256), r(8, 64, 256), r(8, 64, 256), r(8, 256, 64), r(8, 256)
layer = DenseMoeLayer(g, u, d, top_k=2)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    a, b = linear(x, w), gated_linear(x, w, w)
    c = layer.forward_x(x, wr) if m <= 16 else a
graph.replay()
torch.cuda.synchronize()
assert torch.equal(a, linear(x, w)) and torch.equal(b, gated_linear(x, w, w))
assert m > 16 or torch.equal(c, layer.forward_x(x, wr))
print("same")
"""


@pytest.mark.parametrize("m", [3, 100, 2000])
def test_first_call_in_a_capture(m, cuda_device):
    r = subprocess.run([sys.executable, "-c", CODE, str(m)], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]
