"""Microscaled 4-bit matrices and the dense layer over them (C ABI:
include/xse_mx.h).

A matrix is held as E2M1 codes with one power-of-two scale per 32 elements of
a row (MXFP4): 4.25 bits an element. `linear` multiplies two such matrices on
the tensor cores' 4-bit path, beside the fp32 and split-TF32 layers of
dlrm.py. Tensors are torch CUDA tensors; torch is used only for device memory
and streams.
"""

import contextlib
import ctypes
import functools
from typing import Optional

import torch

from . import _capi as C
from .engine import stream_handle

ACT_NONE, ACT_RELU, ACT_SIGMOID = C.ACT_NONE, C.ACT_RELU, C.ACT_SIGMOID
BLOCK = 32  # elements per scale

_FLOATS = {torch.float32: C.DT_F32, torch.bfloat16: C.DT_BF16}


# Scratch bytes by sizes (a call into the library costs half a microsecond).
_linear_workspace = functools.lru_cache(maxsize=1024)(
    C.lib.xse_linear_mxfp4_workspace)

# The current device's index and the raw cudaStream_t of a device's current
# stream, without building torch objects: a call on a few rows lasts a few
# microseconds, as long as those would take. A torch without these (one without
# CUDA, on which the package's host side still imports) has the public ones.
current_device = getattr(torch._C, "_cuda_getDevice",  # pylint: disable=protected-access
                         torch.cuda.current_device)
current_stream = getattr(torch._C, "_cuda_getCurrentRawStream",  # pylint: disable=protected-access
                         lambda index: torch.cuda.current_stream(
                             index).cuda_stream)


def invalid(message):
  return C.XseError(C.INVALID_ARGUMENT, message)


MOST_INT = 2 ** 31 - 1  # of the C ABI's 32-bit sizes; ctypes would cut larger ones


def float_code(t, what):
  """XSE_DT_* of a float32 or bfloat16 CUDA tensor."""
  code = _FLOATS.get(t.dtype)
  if code is None:
    raise invalid(f"{what} must be float32 or bfloat16, got {t.dtype}")
  if not t.is_cuda:
    raise invalid(f"{what} must be a CUDA tensor")
  return code


def matrix(t, what, rows=None):
  """(XSE_DT_*, rows, columns, row stride) of a 2-D float32 or bfloat16 CUDA
  tensor whose rows are contiguous (and as many as `rows`, if given)."""
  code = float_code(t, what)
  shape = t.shape
  if len(shape) != 2:
    raise invalid(f"{what} must be 2-D, got shape {tuple(shape)}")
  n, cols = shape
  if rows is not None and n != rows:
    raise invalid(f"{what} must have {rows} rows, got shape {tuple(shape)}")
  if cols > MOST_INT:
    raise invalid(f"{what} has {cols} columns: less than 2^31 are served")
  stride, step = t.stride()
  if cols > 1 and step != 1:
    raise invalid(f"{what} needs unit column stride")
  if n <= 1:
    return code, n, cols, max(cols, 1)
  if stride < cols:
    raise invalid(f"{what} needs a row stride of at least its columns")
  return code, n, cols, stride


def new_like(device, size, dtype):
  """`size` elements on a device, or on that of a tensor."""
  if isinstance(device, torch.Tensor):
    return device.new_empty(size, dtype=dtype)
  return torch.empty(size, dtype=dtype, device=device)


@contextlib.contextmanager
def on(index, stream):
  """Makes a device and (if given) a stream of it current. A call for another
  device or stream than the current ones makes itself again within: its scratch
  and outputs then come from that stream's pool."""
  if index < 0:
    raise invalid("tensors must be on a CUDA device")
  if stream is not None and stream.device.index != index:
    raise invalid(f"a stream of {stream.device} for tensors on device {index}")
  with torch.cuda.device(index):
    if stream is None:
      yield
    else:
      with torch.cuda.stream(stream):
        yield


def same_device(index, *tensors):
  """Refuses a call whose tensors do not all lie on device `index`."""
  for t in tensors:
    if t is not None and t.get_device() != index:
      raise invalid(f"tensors on {t.device} and device {index} in one call")


def _matrix_sizes(rows, cols, groups):
  """Refuses the sizes of a 4-bit matrix that are not served."""
  if not (0 <= rows <= MOST_INT and 1 <= cols <= 2 ** 30 and
          1 <= groups <= MOST_INT):
    raise invalid("4-bit matrix needs 0 <= rows < 2^31, 1 <= cols <= 2^30 "
                  "and 1 <= groups < 2^31.")


class MxMatrix:
  """`groups` matrices of [rows, cols] in 4 bits (xse_mx_matrix): codes and
  scales are uint8 tensors of xse_mxfp4_codes_bytes and
  xse_mxfp4_scales_bytes."""

  __slots__ = ("_codes", "_scales", "_at", "rows", "cols", "groups", "index",
               "ref")

  def __init__(self, codes, scales, rows, cols, groups=1):
    _matrix_sizes(rows, cols, groups)
    for name, t, need in (
        ("codes", codes, C.lib.xse_mxfp4_codes_bytes(rows, cols, groups)),
        ("scales", scales, C.lib.xse_mxfp4_scales_bytes(rows, cols, groups))):
      if rows > 0 and need == 0:
        raise invalid("4-bit matrix needs less than 2^63 bytes")
      if t.dtype != torch.uint8 or not t.is_contiguous() or \
          t.numel() < need or not t.is_cuda:
        raise invalid(f"4-bit matrix {name}: {need} contiguous uint8 bytes on "
                      f"a CUDA device needed, got {t.numel()} of {t.dtype}")
    if codes.device != scales.device:
      raise invalid("4-bit matrix: codes and scales on one device")
    self._codes, self._scales, self._at = codes, scales, None
    self._set(codes.data_ptr(), scales.data_ptr(), rows, cols, groups)

  def _set(self, codes, scales, rows, cols, groups):
    self.rows, self.cols, self.groups = rows, cols, groups
    self.index = self._codes.get_device()
    self.ref = ctypes.byref(C.MxMatrixStruct(codes, scales, rows, cols,
                                             groups))

  @property
  def codes(self):
    return self._codes if self._at is None else self._codes[:self._at]

  @property
  def scales(self):
    return self._scales if self._at is None else self._codes[self._at:]

  @property
  def device(self):
    return self._codes.device

  def get_device(self):
    return self.index

  dtype = torch.uint8

  def new_empty(self, *shape, dtype=torch.uint8):
    """A tensor on the matrix's device."""
    return self._codes.new_empty(*shape, dtype=dtype)

  @classmethod
  def empty(cls, rows, cols, groups=1, device="cuda"):
    """A matrix to be filled, on a device or that of a tensor; codes and scales
    share one allocation."""
    _matrix_sizes(rows, cols, groups)
    at = groups * rows * ((cols + 31) // 32 * 16)  # a multiple of 16
    self = cls.__new__(cls)
    size = at + groups * ((rows + 127) // 128) * ((cols + 127) // 128) * 512
    self._codes = new_like(device, size, torch.uint8)
    self._scales, self._at = None, at
    start = self._codes.data_ptr()
    self._set(start, start + at if start else 0, rows, cols, groups)
    return self


def quantize(x, out: Optional[MxMatrix] = None, *, stream=None) -> MxMatrix:
  """x ([rows, cols] or [groups, rows, cols], float32 or bfloat16, any
  strides) as an MxMatrix; blocks of 32 run along the last axis. A layer's
  [in, out] kernel is quantised as `quantize(kernel.t())`."""
  code = float_code(x, "x")
  index = x.get_device()
  if stream is not None or index != current_device():
    with on(index, stream):
      return quantize(x, out)
  shape, strides = x.shape, x.stride()
  if len(shape) == 2:
    groups, (rows, cols), group_stride = 1, shape, 0
  elif len(shape) == 3:
    groups, rows, cols = shape
    group_stride = strides[0]
  else:
    raise invalid(f"x must be 2-D or 3-D, got shape {tuple(shape)}")
  if out is None:
    out = MxMatrix.empty(rows, cols, groups, x)
  elif (out.rows, out.cols, out.groups) != (rows, cols, groups):
    raise invalid(f"out holds {out.groups} x {out.rows} x {out.cols}, x has "
                  f"shape {tuple(shape)}")
  if out.index != index:
    same_device(index, out)
  C.check(C.lib.xse_mxfp4_quantize(
      x.data_ptr(), code, group_stride, strides[-2], strides[-1], out.ref,
      current_stream(index)))
  return out


def dequantize(q: MxMatrix, out=None, *, dtype=torch.float32, stream=None):
  """The values q stands for, [rows, cols] ([groups, rows, cols] for several
  groups), in float32 or bfloat16 (exact in both)."""
  index = q.index
  if stream is not None or index != current_device():
    with on(index, stream):
      return dequantize(q, out, dtype=dtype)
  shape = (q.rows, q.cols) if q.groups == 1 else (q.groups, q.rows, q.cols)
  if out is None:
    out = q.new_empty(*shape, dtype=dtype)
  else:
    same_device(index, out)
    if out.shape != shape:
      raise invalid(f"out has shape {tuple(out.shape)}, not {shape}")
  if q.groups == 1:
    group_stride, (code, _, _, stride) = 0, matrix(out, "out")
  else:
    group_stride, (code, _, _, stride) = out.stride(0), matrix(out[0], "out")
    if group_stride == 0:
      raise invalid("out's groups need places of their own")
  C.check(C.lib.xse_mxfp4_dequantize(q.ref, out.data_ptr(), code, group_stride,
                                     stride, current_stream(index)))
  return out


def bias_pointer(bias, shape):
  """Pointer of a float32 bias of `shape`, None without one."""
  if bias is None:
    return None
  if bias.dtype != torch.float32 or bias.shape != shape or \
      not bias.is_contiguous():
    raise invalid(f"bias must be contiguous float32 of shape {shape}, got "
                  f"{bias.dtype} {tuple(bias.shape)}")
  return bias.data_ptr()


def layer_output(out, like, rows, cols, dtype):
  """(tensor, XSE_DT_*, row stride) of a layer's [rows, cols] output, a new one
  of `like`'s device without `out`."""
  if out is None:
    if like.dtype == dtype:
      return like.new_empty(rows, cols), _FLOATS[dtype], cols
    return like.new_empty(rows, cols, dtype=dtype), _FLOATS[dtype], cols
  if out.shape != (rows, cols):
    raise invalid(f"out has shape {tuple(out.shape)}, not {(rows, cols)}")
  code, _, _, stride = matrix(out, "out")
  return out, code, stride


def linear(x, w: MxMatrix, bias=None, activation=ACT_NONE, out=None, *,
           stream=None):
  """out = act(Q(x) W^T + bias) for x [rows, in] (float32 or bfloat16, or an
  MxMatrix already quantised) and w [out, in]; Q is `quantize`. Accumulated
  in fp32 and rounded once to out's type (x's by default; float32 for an
  MxMatrix). out may not share elements with x."""
  index = w.index
  if stream is not None or index != current_device():
    with on(index, stream):
      return linear(x, w, bias, activation, out)
  same_device(index, x, bias, out)
  bias_ptr = bias_pointer(bias, (w.rows,))
  if isinstance(x, MxMatrix):
    out, out_code, out_stride = layer_output(out, w, x.rows, w.rows,
                                             torch.float32)
    C.check(C.lib.xse_linear_forward_mxfp4_q(
        x.ref, w.ref, bias_ptr, activation, out.data_ptr(), out_code,
        out_stride, current_stream(index)))
    return out
  code, rows, cols, x_stride = matrix(x, "x")
  if cols != w.cols:
    raise invalid(f"x has {cols} columns, w {w.cols}")
  out, out_code, out_stride = layer_output(out, x, rows, w.rows, x.dtype)
  size = _linear_workspace(rows, cols)
  scratch = w.new_empty(size) if size else None
  C.check(C.lib.xse_linear_forward_mxfp4(
      x.data_ptr(), code, rows, x_stride, w.ref, bias_ptr, activation,
      out.data_ptr(), out_code, out_stride,
      scratch.data_ptr() if size else None, size, current_stream(index)))
  return out


def check(stream=None):
  """Waits for the stream (the current one by default); raises if a product's
  kernel on its device gave up a wait."""
  if stream is None:
    C.check(C.lib.xse_mxfp4_check(stream_handle()))
    return
  with torch.cuda.device(stream.device):
    C.check(C.lib.xse_mxfp4_check(stream_handle(stream)))
