"""The math modes of the DLRM tower's layers, on the CPU: its own modes leave
the layers that they do not serve in fp32, all others reach the library, which
refuses the unknown ones before it touches the device."""

import types

import pytest
import torch


def tower(xse, math):
  return xse.dlrm.DenseTower(num_dense=13, num_tables=2, dim=8, bottom=(8,),
                             top=(4, 1), device="cpu", math=math)


def layer_math(xse, monkeypatch, math):
  """The modes in which a tower of `math` runs its layers."""
  seen = []
  monkeypatch.setattr(
      xse.dlrm, "linear",
      lambda x, layer, out, *, math, stream: seen.append(math) or out)
  t = tower(xse, xse._capi.MATH_FP32)
  t.math = math
  t.bottom_forward(torch.zeros(3, 13))
  t.top_forward(torch.zeros(3, t.width_stride))
  assert len(seen) == 3
  return set(seen)


def test_modes_that_reach_the_library(xse, monkeypatch):
  C, dlrm = xse._capi, xse.dlrm
  for math in (C.MATH_FP32, C.MATH_BF16X9, C.MATH_TF32, 5, 7, -1):
    assert layer_math(xse, monkeypatch, math) == {math}
  for math in (dlrm.MATH_TF32X3, dlrm.MATH_MXFP4):
    assert layer_math(xse, monkeypatch, math) == {C.MATH_FP32}


@pytest.mark.parametrize("math", [5, 7, -1])
def test_unknown_modes_are_refused(xse, math):
  with pytest.raises(xse.XseError, match="Unknown GEMM math mode") as e:
    tower(xse, math).bottom_forward(torch.zeros(3, 13),
                                    stream=types.SimpleNamespace(cuda_stream=0))
  assert e.value.code == xse._capi.INVALID_ARGUMENT
