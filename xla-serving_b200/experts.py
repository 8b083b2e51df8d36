"""Rows sorted by expert and back, and the experts' 4-bit dense layers (C ABI:
include/xse_experts.h).

A mixture of experts for one batch:

  plan = experts.sort(ids, num_experts)          # ids [tokens, topk]
  h = experts.linear(x, plan, w1, b1, mx.ACT_RELU)         # sorted rows
  y = experts.linear(h, plan, w2, b2, sorted_rows=True)
  out = experts.combine(y, plan, weights)        # weights [tokens, topk]

`gather` gives the sorted rows themselves, for experts computed elsewhere;
`combine_backward` and `combine` without weights are the gradients of
`combine` and `gather`. Outputs may not share elements with inputs.
"""

import ctypes
import functools

import torch

from . import _capi as C
from .mx import (ACT_NONE, MOST_INT, MxMatrix, bias_pointer, current_device,
                 current_stream, invalid, layer_output, matrix, new_like, on,
                 same_device)

MAX_EXPERTS = 1024
_sort_workspace = functools.lru_cache(maxsize=1024)(
    C.lib.xse_expert_sort_workspace)
_linear_workspace = functools.lru_cache(maxsize=1024)(
    C.lib.xse_expert_linear_workspace)
_INDEX = {torch.int32: C.INDEX_I32, torch.int64: C.INDEX_I64}


def _plan_sizes(tokens, topk, num_experts):
  """Refuses the sizes of a plan that are not served."""
  if topk < 1 or topk > MOST_INT or not 1 <= num_experts <= MAX_EXPERTS:
    raise invalid(f"an expert plan needs topk >= 1 and 1 to {MAX_EXPERTS} "
                  "experts")
  if tokens * topk > MOST_INT:
    raise invalid("an expert plan holds less than 2^31 pairs")


class ExpertPlan:
  """(token, choice) pairs sorted by expert (xse_expert_plan), int32:
  offsets [num_experts + 1], order [tokens * topk] (pair of each sorted row,
  -1 behind the last), slots [tokens, topk] (sorted row of each pair, -1 for
  a dropped one)."""

  __slots__ = ("_offsets", "_order", "_slots", "_buffer", "tokens", "topk",
               "pairs", "num_experts", "shape", "index", "ref")

  def __init__(self, offsets, order, slots):
    for name, t in (("offsets", offsets), ("order", order), ("slots", slots)):
      if t.dtype != torch.int32 or not t.is_cuda or not t.is_contiguous():
        raise invalid(f"plan.{name} must be a contiguous int32 CUDA tensor")
    if slots.dim() != 2 or order.numel() != slots.numel() or \
        offsets.numel() < 2:
      raise invalid("a plan has slots [tokens, topk], order [tokens * topk] "
                    "and offsets [num_experts + 1]")
    _plan_sizes(*slots.shape, offsets.numel() - 1)
    if not offsets.device == order.device == slots.device:
      raise invalid("a plan's tensors lie on one device")
    self._offsets, self._order, self._slots = offsets, order, slots
    self._buffer = slots
    self._set(offsets.data_ptr(), order.data_ptr(), slots.data_ptr(),
              *slots.shape, offsets.numel() - 1)

  def _set(self, offsets, order, slots, tokens, topk, num_experts):
    self.tokens, self.topk, self.num_experts = tokens, topk, num_experts
    self.pairs = tokens * topk
    self.shape = (tokens, topk)  # of ids, slots and weights
    self.index = self._buffer.get_device()
    self.ref = ctypes.byref(C.ExpertPlanStruct(offsets, order, slots, tokens,
                                               topk, num_experts))

  def _view(self, shape, strides, at):
    return torch.as_strided(self._buffer, shape, strides, at)

  @property
  def slots(self):
    if self._slots is None:
      self._slots = self._view((self.tokens, self.topk), (self.topk, 1), 0)
    return self._slots

  @property
  def order(self):
    if self._order is None:
      self._order = self._view((self.pairs,), (1,), _quads(self.pairs))
    return self._order

  @property
  def offsets(self):
    if self._offsets is None:
      self._offsets = self._view((self.num_experts + 1,), (1,),
                                 2 * _quads(self.pairs))
    return self._offsets

  @property
  def device(self):
    return self._buffer.device

  def get_device(self):
    return self.index

  @classmethod
  def empty(cls, tokens, topk, num_experts, device="cuda"):
    """A plan to be filled, on a device or that of a tensor; its arrays (slots,
    order, offsets, each on a 16-byte boundary) share one allocation."""
    _plan_sizes(tokens, topk, num_experts)
    part = _quads(tokens * topk)
    self = cls.__new__(cls)
    self._buffer = new_like(device, 2 * part + num_experts + 1, torch.int32)
    self._offsets = self._order = self._slots = None
    start = self._buffer.data_ptr()
    self._set(start + 8 * part, start + 4 * part, start, tokens, topk,
              num_experts)
    return self


def _quads(n):
  """n rounded up to whole 16-byte quads of int32."""
  return (n + 3) // 4 * 4


def sort(ids, num_experts, plan=None, *, stream=None) -> ExpertPlan:
  """The plan of ids [tokens, topk] (int32 or int64): pairs by expert, those
  of one expert in their order. A pair whose id lies outside [0, num_experts)
  is dropped (padding rows are given -1)."""
  code = _INDEX.get(ids.dtype)
  if code is None or ids.dim() != 2 or not ids.is_cuda or \
      not ids.is_contiguous():
    raise invalid("expert ids must be a contiguous 2-D int32 or int64 CUDA "
                  f"tensor, got {ids.dtype} {tuple(ids.shape)}")
  index = ids.get_device()
  if stream is not None or index != current_device():
    with on(index, stream):
      return sort(ids, num_experts, plan)
  tokens, topk = ids.shape
  if plan is None:
    plan = ExpertPlan.empty(tokens, topk, num_experts, ids)
  elif (plan.tokens, plan.topk, plan.num_experts) != (tokens, topk,
                                                      num_experts):
    raise invalid("the plan has other sizes than ids")
  same_device(index, plan)
  size = _sort_workspace(plan.pairs, num_experts)
  scratch = ids.new_empty(size, dtype=torch.uint8) if size else None
  C.check(C.lib.xse_expert_sort(
      ids.data_ptr(), code, plan.ref, scratch.data_ptr() if size else None,
      size, current_stream(index)))
  return plan


def _weights(weights, plan):
  if weights is None:
    return None
  if weights.dtype != torch.float32 or weights.shape != plan.shape or \
      not weights.is_contiguous():
    raise invalid(f"weights must be contiguous float32 of shape {plan.shape}, "
                  f"got {weights.dtype} {tuple(weights.shape)}")
  if weights.get_device() != plan.index:
    same_device(plan.index, weights)
  return weights.data_ptr()


def _output(out, rows, cols, like, what="out"):
  """(tensor, row stride) of an output of `like`'s type."""
  if out is None:
    return like.new_empty(rows, cols), cols
  same_device(like.get_device(), out)
  if out.shape != (rows, cols) or out.dtype != like.dtype:
    raise invalid(f"{what} must be {like.dtype} of shape {(rows, cols)}, got "
                  f"{out.dtype} {tuple(out.shape)}")
  return out, matrix(out, what)[3]


def gather(x, plan: ExpertPlan, out=None, *, stream=None):
  """x's rows in sorted order: out[r] = x[plan.order[r] // topk], zeros behind
  the last sorted row. Its gradient is combine(grad, plan)."""
  index = x.get_device()
  if stream is not None or index != current_device():
    with on(index, stream):
      return gather(x, plan, out)
  if plan.index != index:
    same_device(index, plan)
  code, _, cols, stride = matrix(x, "x", plan.tokens)
  out, out_stride = _output(out, plan.pairs, cols, x)
  C.check(C.lib.xse_expert_gather(
      x.data_ptr(), code, cols, stride, plan.ref, out.data_ptr(), out_stride,
      current_stream(index)))
  return out


def combine(y, plan: ExpertPlan, weights=None, out=None, *, stream=None):
  """out[t] = sum over j of weights[t, j] * y[plan.slots[t, j]] (weights 1
  without them), summed in fp32 in the order of the choices; a row all of
  whose pairs were dropped is zero."""
  index = y.get_device()
  if stream is not None or index != current_device():
    with on(index, stream):
      return combine(y, plan, weights, out)
  if plan.index != index:
    same_device(index, plan)
  code, _, cols, stride = matrix(y, "y", plan.pairs)
  w = _weights(weights, plan)
  out, out_stride = _output(out, plan.tokens, cols, y)
  C.check(C.lib.xse_expert_combine(
      y.data_ptr(), code, cols, stride, plan.ref, w, out.data_ptr(),
      out_stride, current_stream(index)))
  return out


def combine_backward(grad, y, plan: ExpertPlan, weights=None, grad_y=None,
                     grad_weights=None, *, stream=None):
  """(grad_y, grad_weights) of combine for grad [tokens, cols]: sorted row r
  of pair p gets weights[p] * grad[p // topk] (zeros behind the last), weight
  (t, j) the dot product of grad[t] and its sorted row (0 for a dropped
  pair)."""
  index = y.get_device()
  if stream is not None or index != current_device():
    with on(index, stream):
      return combine_backward(grad, y, plan, weights, grad_y, grad_weights)
  if plan.index != index:
    same_device(index, plan)
  code, _, cols, y_stride = matrix(y, "y", plan.pairs)
  grad_code, _, grad_cols, grad_stride = matrix(grad, "grad", plan.tokens)
  same_device(index, grad)
  if grad_code != code or grad_cols != cols:
    raise invalid("grad and y need one type and width")
  w = _weights(weights, plan)
  grad_y, gy_stride = _output(grad_y, plan.pairs, cols, y, "grad_y")
  if grad_weights is None:
    grad_weights = y.new_empty(plan.tokens, plan.topk, dtype=torch.float32)
  C.check(C.lib.xse_expert_combine_backward(
      grad.data_ptr(), y.data_ptr(), code, cols, grad_stride, y_stride,
      plan.ref, w, grad_y.data_ptr(), gy_stride, _weights(grad_weights, plan),
      current_stream(index)))
  return grad_y, grad_weights


def linear(x, plan: ExpertPlan, w: MxMatrix, bias=None, activation=ACT_NONE,
           out=None, *, sorted_rows=False, stream=None):
  """Each sorted row's product with its expert's weights: out[r] =
  act(Q(x_r) W_e^T + bias_e), zeros behind the last sorted row. x is [tokens,
  in] in the tokens' order, or [tokens * topk, in] with sorted_rows; w holds
  num_experts groups of [out, in], bias is [num_experts, out]. out is
  [tokens * topk, out] of x's type by default."""
  index = x.get_device()
  if stream is not None or index != current_device():
    with on(index, stream):
      return linear(x, plan, w, bias, activation, out,
                    sorted_rows=sorted_rows)
  same_device(index, plan, w, bias, out)
  code, _, cols, stride = matrix(
      x, "x", plan.pairs if sorted_rows else plan.tokens)
  if cols != w.cols:
    raise invalid(f"x has {cols} columns, w {w.cols}")
  bias_ptr = bias_pointer(bias, (w.groups, w.rows))
  out, out_code, out_stride = layer_output(out, x, plan.pairs, w.rows, x.dtype)
  size = _linear_workspace(plan.pairs, plan.num_experts, cols)
  scratch = w.new_empty(size) if size else None
  C.check(C.lib.xse_expert_linear_mxfp4(
      x.data_ptr(), code, stride, 1 if sorted_rows else 0, plan.ref, w.ref,
      bias_ptr, activation, out.data_ptr(), out_code, out_stride,
      scratch.data_ptr() if size else None, size,
      current_stream(index)))
  return out
