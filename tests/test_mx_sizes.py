"""Sizes that the C ABI's 32-bit fields would cut, on the CPU with stand-ins
for tensors: a call that they reach is refused, not served in part."""

import types

import pytest
import torch


def tensor(shape, dtype=torch.bfloat16, strides=None):
  """What the argument checks ask of a contiguous CUDA tensor."""
  count = 1
  for n in shape:
    count *= n
  if strides is None:
    strides, step = [], 1
    for n in reversed(shape):
      strides.insert(0, step)
      step *= n
  return types.SimpleNamespace(
      shape=torch.Size(shape), dtype=dtype, is_cuda=True, device="cuda:0",
      stride=lambda: tuple(strides), numel=lambda: count,
      dim=lambda: len(shape), is_contiguous=lambda: True,
      data_ptr=lambda: 4096, get_device=lambda: 0)


def refused(xse, word, call):
  with pytest.raises(xse.XseError, match=word) as e:
    call()
  assert e.value.code == xse._capi.INVALID_ARGUMENT


@pytest.mark.parametrize("cols", [2 ** 31, 2 ** 32 + 64])
def test_wide_rows(xse, cols):
  refused(xse, "columns", lambda: xse.mx.matrix(tensor((1, cols)), "x"))


def test_rows_that_fit(xse):
  code, rows, cols, stride = xse.mx.matrix(tensor((2 ** 33, 2 ** 31 - 1)), "x")
  assert (code, rows, cols, stride) == (xse._capi.DT_BF16, 2 ** 33,
                                        2 ** 31 - 1, 2 ** 31 - 1)


@pytest.mark.parametrize("rows,cols,groups", [
    (-1, 64, 1), (2 ** 31, 64, 1), (1, 0, 1), (1, 2 ** 30 + 1, 1),
    (1, 2 ** 32 + 64, 1), (1, 64, 0), (1, 64, 2 ** 32 + 1)])
def test_4_bit_matrices(xse, rows, cols, groups):
  buffer = tensor((4096,), torch.uint8)
  refused(xse, "4-bit matrix needs",
          lambda: xse.mx.MxMatrix(buffer, buffer, rows, cols, groups))
  refused(xse, "4-bit matrix needs",
          lambda: xse.mx.MxMatrix.empty(rows, cols, groups, "cpu"))


def test_matrices_that_fit(xse):
  buffer = tensor((4096,), torch.uint8)
  assert xse.mx.MxMatrix(buffer, buffer, 3, 64, 2).cols == 64
  assert xse.mx.MxMatrix.empty(0, 64, 1, "cpu").rows == 0


@pytest.mark.parametrize("tokens,topk,experts,word", [
    (1, 2 ** 32 + 8, 4, "topk"), (2 ** 30, 2, 4, "pairs"),
    (2 ** 31, 1, 4, "pairs"), (4, 0, 4, "topk"), (4, 2, 1025, "experts")])
def test_plans(xse, tokens, topk, experts, word):
  i32 = torch.int32
  refused(xse, word, lambda: xse.experts.ExpertPlan(
      tensor((experts + 1,), i32), tensor((tokens * topk,), i32),
      tensor((tokens, topk), i32)))
  refused(xse, word,
          lambda: xse.experts.ExpertPlan.empty(tokens, topk, experts, "cpu"))


def test_plans_that_fit(xse):
  i32 = torch.int32
  plan = xse.experts.ExpertPlan(tensor((5,), i32), tensor((2 ** 31 - 1,), i32),
                                tensor((2 ** 31 - 1, 1), i32))
  assert plan.pairs == 2 ** 31 - 1 and plan.num_experts == 4
