"""The library without the extension that generation's calls go through."""
from __future__ import annotations

import os
import subprocess
import sys

from conftest import PKG

CODE = r"""
import sys
sys.modules["lzhip._torchcall"] = None  # an import of it fails
from lzhip import _lib, ops
assert _lib.load().lz_version() == 1 and _lib.query("lz_gemm_plan", 256, 256, 256, 0, 0) >= 0
import torch
for call in (lambda: _lib.tensor_calls(), lambda: ops.process_logits(torch.zeros(1, 2))):
    for _ in range(2):
        try:
            call()
        except _lib.HipLibraryError as e:
            assert "_torchcall" in str(e) and "build.py" in str(e), e
        else:
            raise SystemExit("not refused")
print("fine")
"""


def test_training_loads_without_the_tensor_calls():
    ran = subprocess.run([sys.executable, "-c", CODE], env=dict(os.environ, PYTHONPATH=PKG), capture_output=True, text=True)
    assert ran.returncode == 0 and "fine" in ran.stdout, ran.stderr
