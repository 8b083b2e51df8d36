"""The package on a torch without CUDA bindings: it imports, and its calls
refuse host tensors as they do elsewhere."""

import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = """
import sys
import torch
for name in ("_cuda_getDevice", "_cuda_getCurrentRawStream"):
  if hasattr(torch._C, name):
    delattr(torch._C, name)
sys.path.insert(0, sys.argv[1])
from tests.conftest import load_package
xse = load_package()
assert xse._capi.lib.xse_mxfp4_codes_bytes(1, 32, 1) == 16
for call in (lambda: xse.mx.quantize(torch.zeros(2, 32)),
             lambda: xse.experts.sort(torch.zeros((2, 1), dtype=torch.int32), 3)):
  try:
    call()
  except xse.XseError as e:
    assert e.code == xse._capi.INVALID_ARGUMENT
  else:
    raise AssertionError("a host tensor was taken")
print("imported")
"""


def test_import_without_cuda_bindings():
  done = subprocess.run([sys.executable, "-c", PROGRAM, ROOT],
                        capture_output=True, text=True, check=False)
  assert done.returncode == 0, done.stderr
  assert "imported" in done.stdout
