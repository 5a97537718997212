"""The package imports, and plans, with a torch that was built without CUDA."""

import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent.parent / "quant-studio_b200"

PROGRAM = """
import sys, torch
for name in [n for n in dir(torch._C) if n.startswith("_cuda_")]:
    delattr(torch._C, name)  # as in such a build
sys.path.insert(0, sys.argv[1])
import kernels
from kernels import _native, ops
assert "Q4_K" in {str(k).upper().split(".")[-1] for k in kernels.QUANT_TYPES}
try:
    ops.route(torch.zeros(2, 8), 2)
except _native.QsError as e:
    assert e.code == _native.QS_EINVAL
else:
    raise AssertionError("a CPU tensor was taken")
"""


def test_import():
    r = subprocess.run([sys.executable, "-c", PROGRAM, str(PKG)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
