"""Microscaled 4-bit matrices and the dense layer over them (C ABI:
include/xse_mx.h).

A matrix is held as E2M1 codes with one power-of-two scale per 32 elements of
a row (MXFP4): 4.25 bits an element. `linear` multiplies two such matrices on
the tensor cores' 4-bit path, beside the fp32 and split-TF32 layers of
dlrm.py. Tensors are torch CUDA tensors; torch is used only for device memory
and streams.
"""

import ctypes
import dataclasses
from typing import Optional

import torch

from . import _capi as C
from .engine import stream_handle

ACT_NONE, ACT_RELU, ACT_SIGMOID = C.ACT_NONE, C.ACT_RELU, C.ACT_SIGMOID
BLOCK = 32  # elements per scale

_FLOATS = {torch.float32: C.DT_F32, torch.bfloat16: C.DT_BF16}


def invalid(message):
  return C.XseError(C.INVALID_ARGUMENT, message)


def float_code(t, what):
  """XSE_DT_* of a float32 or bfloat16 CUDA tensor."""
  code = _FLOATS.get(t.dtype)
  if code is None:
    raise invalid(f"{what} must be float32 or bfloat16, got {t.dtype}")
  if not t.is_cuda:
    raise invalid(f"{what} must be a CUDA tensor")
  return code


def row_stride(t, what):
  """Row stride of a 2-D tensor whose rows are contiguous."""
  if t.dim() != 2:
    raise invalid(f"{what} must be 2-D, got shape {tuple(t.shape)}")
  rows, cols = t.shape
  if cols > 1 and t.stride(1) != 1:
    raise invalid(f"{what} needs unit column stride")
  if rows > 1:
    if t.stride(0) < cols:
      raise invalid(f"{what} needs a row stride of at least its columns")
    return t.stride(0)
  return max(cols, 1)


class On:
  """The device and stream of one call: makes `device` current for the C call
  and allocates from the given stream's pool. Every tensor of the call must
  lie on the device."""

  __slots__ = ("device", "stream", "_device", "_stream")

  def __init__(self, device, stream, *tensors):
    for t in tensors:
      if t is not None and t.device != device:
        raise invalid(f"tensors on {t.device} and {device} in one call")
    if stream is not None and stream.device != device:
      raise invalid(f"a stream of {stream.device} for tensors on {device}")
    self.device, self.stream = device, stream
    self._device = self._stream = None

  def __enter__(self):
    if torch.cuda.current_device() != self.device.index:
      self._device = torch.cuda.device(self.device)
      self._device.__enter__()
    if self.stream is not None:
      self._stream = torch.cuda.stream(self.stream)
      self._stream.__enter__()
    return stream_handle(self.stream)

  def __exit__(self, *exc):
    if self._stream is not None:
      self._stream.__exit__(*exc)
    if self._device is not None:
      self._device.__exit__(*exc)


@dataclasses.dataclass
class MxMatrix:
  """`groups` matrices of [rows, cols] in 4 bits (xse_mx_matrix)."""

  codes: torch.Tensor   # uint8, xse_mxfp4_codes_bytes
  scales: torch.Tensor  # uint8, xse_mxfp4_scales_bytes
  rows: int
  cols: int
  groups: int = 1

  def __post_init__(self):
    for name, t, need in (
        ("codes", self.codes,
         C.lib.xse_mxfp4_codes_bytes(self.rows, self.cols, self.groups)),
        ("scales", self.scales,
         C.lib.xse_mxfp4_scales_bytes(self.rows, self.cols, self.groups))):
      if t.dtype != torch.uint8 or not t.is_contiguous() or t.numel() < need:
        raise invalid(f"4-bit matrix {name}: {need} contiguous uint8 bytes "
                      f"needed, got {t.numel()} of {t.dtype}")
    if self.codes.device != self.scales.device:
      raise invalid("4-bit matrix: codes and scales on one device")
    self.struct = C.MxMatrixStruct(self.codes.data_ptr(),
                                   self.scales.data_ptr(), self.rows,
                                   self.cols, self.groups)

  @property
  def device(self):
    return self.codes.device

  @classmethod
  def empty(cls, rows, cols, groups=1, device="cuda"):
    if rows < 0 or rows >= 2 ** 31 or cols < 1 or groups < 1:
      raise invalid("4-bit matrix needs 0 <= rows < 2^31, cols >= 1 and "
                    "groups >= 1.")
    codes, scales = (
        torch.empty(f(rows, cols, groups), dtype=torch.uint8, device=device)
        for f in (C.lib.xse_mxfp4_codes_bytes, C.lib.xse_mxfp4_scales_bytes))
    return cls(codes, scales, rows, cols, groups)


def quantize(x, out: Optional[MxMatrix] = None, *, stream=None) -> MxMatrix:
  """x ([rows, cols] or [groups, rows, cols], float32 or bfloat16, any
  strides) as an MxMatrix; blocks of 32 run along the last axis. A layer's
  [in, out] kernel is quantised as `quantize(kernel.t())`."""
  code = float_code(x, "x")
  if x.dim() not in (2, 3):
    raise invalid(f"x must be 2-D or 3-D, got shape {tuple(x.shape)}")
  groups = x.shape[0] if x.dim() == 3 else 1
  rows, cols = x.shape[-2:]
  with On(x.device, stream, out) as s:
    if out is None:
      out = MxMatrix.empty(rows, cols, groups, x.device)
    elif (out.rows, out.cols, out.groups) != (rows, cols, groups):
      raise invalid(f"out holds {out.groups} x {out.rows} x {out.cols}, x has "
                    f"shape {tuple(x.shape)}")
    C.check(C.lib.xse_mxfp4_quantize(
        x.data_ptr(), code, x.stride(0) if groups > 1 else 0, x.stride(-2),
        x.stride(-1), ctypes.byref(out.struct), s))
  return out


def dequantize(q: MxMatrix, out=None, *, dtype=torch.float32, stream=None):
  """The values q stands for, [rows, cols] ([groups, rows, cols] for several
  groups), in float32 or bfloat16 (exact in both)."""
  with On(q.device, stream, out) as s:
    shape = (q.rows, q.cols) if q.groups == 1 else (q.groups, q.rows, q.cols)
    if out is None:
      out = torch.empty(shape, dtype=dtype, device=q.device)
    elif out.shape != shape:
      raise invalid(f"out has shape {tuple(out.shape)}, not {shape}")
    code = float_code(out, "out")
    group = out.stride(0) if q.groups > 1 else 0
    stride = row_stride(out if q.groups == 1 else out[0], "out")
    C.check(C.lib.xse_mxfp4_dequantize(ctypes.byref(q.struct), out.data_ptr(),
                                       code, group, stride, s))
  return out


def check_bias(bias, shape):
  """Pointer of a float32 bias of `shape`, None without one."""
  if bias is None:
    return None
  if bias.dtype != torch.float32 or tuple(bias.shape) != shape or \
      not bias.is_contiguous():
    raise invalid(f"bias must be contiguous float32 of shape {shape}, got "
                  f"{bias.dtype} {tuple(bias.shape)}")
  return bias.data_ptr()


def linear(x, w: MxMatrix, bias=None, activation=ACT_NONE, out=None, *,
           stream=None):
  """out = act(Q(x) W^T + bias) for x [rows, in] (float32 or bfloat16, or an
  MxMatrix already quantised) and w [out, in]; Q is `quantize`. Accumulated
  in fp32 and rounded once to out's type (x's by default; float32 for an
  MxMatrix)."""
  quantised = isinstance(x, MxMatrix)
  if x.device != w.device:
    raise invalid(f"tensors on {x.device} and {w.device} in one call")
  with On(w.device, stream, bias, out) as s:
    rows = x.rows if quantised else x.shape[0]
    if out is None:
      out = torch.empty((rows, w.rows), device=w.device,
                        dtype=torch.float32 if quantised else x.dtype)
    elif tuple(out.shape) != (rows, w.rows):
      raise invalid(f"out has shape {tuple(out.shape)}, not "
                    f"{(rows, w.rows)}")
    out_code = float_code(out, "out")
    out_stride = max(row_stride(out, "out"), w.rows)
    bias_ptr = check_bias(bias, (w.rows,))
    if quantised:
      C.check(C.lib.xse_linear_forward_mxfp4_q(
          ctypes.byref(x.struct), ctypes.byref(w.struct), bias_ptr, activation,
          out.data_ptr(), out_code, out_stride, s))
      return out
    code = float_code(x, "x")
    stride = row_stride(x, "x")
    if x.shape[1] != w.cols:
      raise invalid(f"x has {x.shape[1]} columns, w {w.cols}")
    size = C.lib.xse_linear_mxfp4_workspace(rows, w.cols)
    scratch = torch.empty(size, dtype=torch.uint8, device=w.device)
    C.check(C.lib.xse_linear_forward_mxfp4(
        x.data_ptr(), code, rows, stride, ctypes.byref(w.struct), bias_ptr,
        activation, out.data_ptr(), out_code, out_stride, scratch.data_ptr(),
        size, s))
  return out


def check(stream=None):
  """Waits for the stream; raises if a product's kernel gave up a wait."""
  C.check(C.lib.xse_mxfp4_check(stream_handle(stream)))
