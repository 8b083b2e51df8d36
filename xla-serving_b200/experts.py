"""Rows sorted by expert and back, and the experts' 4-bit dense layers (C ABI:
include/xse_experts.h).

A mixture of experts for one batch:

  plan = experts.sort(ids, num_experts)          # ids [tokens, topk]
  h = experts.linear(x, plan, w1, b1, mx.ACT_RELU)         # sorted rows
  y = experts.linear(h, plan, w2, b2, sorted_rows=True)
  out = experts.combine(y, plan, weights)        # weights [tokens, topk]

`gather` gives the sorted rows themselves, for experts computed elsewhere;
`combine_backward` and `combine` without weights are the gradients of
`combine` and `gather`.
"""

import ctypes
import dataclasses

import torch

from . import _capi as C
from .mx import (ACT_NONE, MxMatrix, On, check_bias, float_code, invalid,
                 row_stride)

MAX_EXPERTS = 1024


@dataclasses.dataclass
class ExpertPlan:
  """(token, choice) pairs sorted by expert (xse_expert_plan), int32:
  offsets [num_experts + 1], order [tokens * topk] (pair of each sorted row,
  -1 behind the last), slots [tokens, topk] (sorted row of each pair, -1 for
  a dropped one)."""

  offsets: torch.Tensor
  order: torch.Tensor
  slots: torch.Tensor

  def __post_init__(self):
    for name in ("offsets", "order", "slots"):
      t = getattr(self, name)
      if t.dtype != torch.int32 or not t.is_cuda or not t.is_contiguous():
        raise invalid(f"plan.{name} must be a contiguous int32 CUDA tensor")
    if self.slots.dim() != 2 or self.order.numel() != self.slots.numel() or \
        self.offsets.numel() < 2:
      raise invalid("a plan has slots [tokens, topk], order [tokens * topk] "
                    "and offsets [num_experts + 1]")
    if not self.offsets.device == self.order.device == self.slots.device:
      raise invalid("a plan's tensors lie on one device")
    self.struct = C.ExpertPlanStruct(
        self.offsets.data_ptr(), self.order.data_ptr(), self.slots.data_ptr(),
        self.tokens, self.topk, self.num_experts)

  @property
  def tokens(self):
    return self.slots.shape[0]

  @property
  def topk(self):
    return self.slots.shape[1]

  @property
  def pairs(self):
    return self.slots.numel()

  @property
  def num_experts(self):
    return self.offsets.numel() - 1

  @property
  def device(self):
    return self.slots.device

  @classmethod
  def empty(cls, tokens, topk, num_experts, device="cuda"):
    if topk < 1 or not 1 <= num_experts <= MAX_EXPERTS:
      raise invalid(f"an expert plan needs topk >= 1 and 1 to {MAX_EXPERTS} "
                    "experts")
    new = lambda *shape: torch.empty(shape, dtype=torch.int32, device=device)  # noqa: E731
    return cls(new(num_experts + 1), new(tokens * topk), new(tokens, topk))


def sort(ids, num_experts, plan=None, *, stream=None) -> ExpertPlan:
  """The plan of ids [tokens, topk] (int32 or int64): pairs by expert, those
  of one expert in their order. A pair whose id lies outside [0, num_experts)
  is dropped (padding rows are given -1)."""
  types = {torch.int32: C.INDEX_I32, torch.int64: C.INDEX_I64}
  if ids.dtype not in types or ids.dim() != 2 or not ids.is_cuda or \
      not ids.is_contiguous():
    raise invalid("expert ids must be a contiguous 2-D int32 or int64 CUDA "
                  f"tensor, got {ids.dtype} {tuple(ids.shape)}")
  with On(ids.device, stream) as s:
    if plan is None:
      plan = ExpertPlan.empty(*ids.shape, num_experts, ids.device)
    elif (plan.tokens, plan.topk, plan.num_experts) != (*ids.shape,
                                                        num_experts) or \
        plan.device != ids.device:
      raise invalid("the plan has other sizes than ids")
    size = C.lib.xse_expert_sort_workspace(plan.pairs, num_experts)
    scratch = torch.empty(size, dtype=torch.uint8, device=ids.device) \
        if size else None
    C.check(C.lib.xse_expert_sort(ids.data_ptr(), types[ids.dtype],
                                  ctypes.byref(plan.struct),
                                  scratch.data_ptr() if size else None, size,
                                  s))
  return plan


def _check_rows(t, rows, what):
  if t.dim() != 2 or t.shape[0] != rows:
    raise invalid(f"{what} must have {rows} rows, got shape {tuple(t.shape)}")


def _check_weights(weights, plan):
  if weights is None:
    return None
  if weights.dtype != torch.float32 or weights.shape != plan.slots.shape or \
      not weights.is_contiguous():
    raise invalid("weights must be contiguous float32 of shape "
                  f"{tuple(plan.slots.shape)}, got {weights.dtype} "
                  f"{tuple(weights.shape)}")
  return weights.data_ptr()


def _output(out, rows, like, what="out"):
  if out is None:
    return torch.empty((rows, like.shape[1]), dtype=like.dtype,
                       device=like.device)
  if tuple(out.shape) != (rows, like.shape[1]) or out.dtype != like.dtype:
    raise invalid(f"{what} must be {like.dtype} of shape "
                  f"{(rows, like.shape[1])}, got {out.dtype} "
                  f"{tuple(out.shape)}")
  return out


def gather(x, plan: ExpertPlan, out=None, *, stream=None):
  """x's rows in sorted order: out[r] = x[plan.order[r] // topk], zeros behind
  the last sorted row. Its gradient is combine(grad, plan)."""
  code = float_code(x, "x")
  _check_rows(x, plan.tokens, "x")
  stride = row_stride(x, "x")
  with On(plan.device, stream, x, out) as s:
    out = _output(out, plan.pairs, x)
    C.check(C.lib.xse_expert_gather(
        x.data_ptr(), code, x.shape[1], stride, ctypes.byref(plan.struct),
        out.data_ptr(), row_stride(out, "out"), s))
  return out


def combine(y, plan: ExpertPlan, weights=None, out=None, *, stream=None):
  """out[t] = sum over j of weights[t, j] * y[plan.slots[t, j]] (weights 1
  without them), summed in fp32 in the order of the choices; a row all of
  whose pairs were dropped is zero."""
  code = float_code(y, "y")
  _check_rows(y, plan.pairs, "y")
  stride = row_stride(y, "y")
  w = _check_weights(weights, plan)
  with On(plan.device, stream, y, weights, out) as s:
    out = _output(out, plan.tokens, y)
    C.check(C.lib.xse_expert_combine(
        y.data_ptr(), code, y.shape[1], stride, ctypes.byref(plan.struct), w,
        out.data_ptr(), row_stride(out, "out"), s))
  return out


def combine_backward(grad, y, plan: ExpertPlan, weights=None, grad_y=None,
                     grad_weights=None, *, stream=None):
  """(grad_y, grad_weights) of combine for grad [tokens, cols]: sorted row r
  of pair p gets weights[p] * grad[p // topk] (zeros behind the last), weight
  (t, j) the dot product of grad[t] and its sorted row (0 for a dropped
  pair)."""
  code = float_code(y, "y")
  _check_rows(y, plan.pairs, "y")
  _check_rows(grad, plan.tokens, "grad")
  if grad.dtype != y.dtype or grad.shape[1] != y.shape[1]:
    raise invalid("grad and y need one type and width")
  w = _check_weights(weights, plan)
  strides = row_stride(grad, "grad"), row_stride(y, "y")
  with On(plan.device, stream, grad, y, weights, grad_y, grad_weights) as s:
    grad_y = _output(grad_y, plan.pairs, y, "grad_y")
    if grad_weights is None:
      grad_weights = torch.empty(plan.slots.shape, dtype=torch.float32,
                                 device=plan.device)
    C.check(C.lib.xse_expert_combine_backward(
        grad.data_ptr(), y.data_ptr(), code, y.shape[1], *strides,
        ctypes.byref(plan.struct), w, grad_y.data_ptr(),
        row_stride(grad_y, "grad_y"), _check_weights(grad_weights, plan), s))
  return grad_y, grad_weights


def linear(x, plan: ExpertPlan, w: MxMatrix, bias=None, activation=ACT_NONE,
           out=None, *, sorted_rows=False, stream=None):
  """Each sorted row's product with its expert's weights: out[r] =
  act(Q(x_r) W_e^T + bias_e), zeros behind the last sorted row. x is [tokens,
  in] in the tokens' order, or [tokens * topk, in] with sorted_rows; w holds
  num_experts groups of [out, in], bias is [num_experts, out]. out is
  [tokens * topk, out] of x's type by default."""
  code = float_code(x, "x")
  _check_rows(x, plan.pairs if sorted_rows else plan.tokens, "x")
  if x.shape[1] != w.cols:
    raise invalid(f"x has {x.shape[1]} columns, w {w.cols}")
  if w.device != plan.device:
    raise invalid(f"tensors on {w.device} and {plan.device} in one call")
  bias_ptr = check_bias(bias, (w.groups, w.rows))
  stride = row_stride(x, "x")
  with On(plan.device, stream, x, bias, out) as s:
    if out is None:
      out = torch.empty((plan.pairs, w.rows), dtype=x.dtype, device=x.device)
    elif tuple(out.shape) != (plan.pairs, w.rows):
      raise invalid(f"out has shape {tuple(out.shape)}, not "
                    f"{(plan.pairs, w.rows)}")
    out_code = float_code(out, "out")
    size = C.lib.xse_expert_linear_workspace(plan.pairs, plan.num_experts,
                                             w.cols)
    scratch = torch.empty(size, dtype=torch.uint8, device=plan.device)
    C.check(C.lib.xse_expert_linear_mxfp4(
        x.data_ptr(), code, stride, 1 if sorted_rows else 0,
        ctypes.byref(plan.struct), ctypes.byref(w.struct), bias_ptr,
        activation, out.data_ptr(), out_code, row_stride(out, "out"),
        scratch.data_ptr(), size, s))
  return out
