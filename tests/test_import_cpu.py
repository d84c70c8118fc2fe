"""The package on a torch that was built without CUDA: everything imports, and calls say what is missing."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CODE = """
import torch
for name in [n for n in dir(torch._C) if n.startswith("_cuda_")]:
    delattr(torch._C, name)
import nano_ktrans_b200 as nk
for name in nk.__all__:
    getattr(nk, name)
x = torch.zeros(2, 8, dtype=torch.bfloat16)
try:
    nk.linear(x, x)
except ValueError as e:
    assert "CUDA" in str(e)
    print("refused")
"""


def test_every_name_imports_without_cuda_bindings():
    r = subprocess.run([sys.executable, "-c", CODE], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "refused" in r.stdout, r.stderr[-2000:]
