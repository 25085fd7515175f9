"""A kernel that a program registers on an op before it imports the package is consulted like one
registered afterwards."""
import os
import subprocess
import sys
from pathlib import Path

PACKAGE = Path(__file__).resolve().parent.parent / "comfy-kitchen_amd"
PROGRAM = """
import torch
lib = torch.library.Library("comfy_kitchen", "FRAGMENT")
lib.impl("quantize_fp8", lambda x, scale, code: x, "CUDA")
lib.impl("paged_attention", lambda *args: args[0], "AutocastCUDA")
from comfy_kitchen.ops import untouched
assert not untouched("quantize_fp8") and not untouched("paged_attention")
assert all(untouched(op) for op in ("dequantize_fp8", "paged_write", "paged_copy", "linear_int4"))
"""


def test_kernels_registered_before_the_import():
    r = subprocess.run([sys.executable, "-c", PROGRAM], env={**os.environ, "PYTHONPATH": str(PACKAGE)},
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
