"""Argument checks of the 4-bit and expert entry points through the C ABI,
without a GPU: every refusal comes before the first CUDA call."""

import ctypes
import types

import numpy as np
import pytest
import torch

from tests import mx_reference as ref


@pytest.fixture(scope="module")
def capi(xse):
  return xse._capi


def refused(capi, rc, *words):
  assert rc == capi.INVALID_ARGUMENT
  for word in words:
    assert word in capi.last_error(), capi.last_error()


def matrix(capi, rows=4, cols=64, groups=1, codes=4096, scales=8192):
  return ctypes.byref(capi.MxMatrixStruct(codes, scales, rows, cols, groups))


def plan(capi, tokens=4, topk=2, experts=3, offsets=4096, order=8192,
         slots=12288):
  return ctypes.byref(capi.ExpertPlanStruct(offsets, order, slots, tokens,
                                            topk, experts))


def test_buffer_sizes(capi):
  lib = capi.lib
  for rows, cols, groups in ((1, 1, 1), (128, 128, 1), (129, 129, 3),
                             (5, 479, 2), (0, 64, 1), (70000, 4096, 1)):
    blocks, tiles = -(-cols // 32), -(-rows // 128) * -(-cols // 128)
    assert lib.xse_mxfp4_codes_bytes(rows, cols, groups) == \
        groups * rows * blocks * 16
    assert lib.xse_mxfp4_scales_bytes(rows, cols, groups) == \
        groups * tiles * 512
    need = lib.xse_linear_mxfp4_workspace(rows, cols)
    assert need == 0 if rows <= 32 else need >= rows * blocks * 16 + tiles * 512
  for rows, cols, groups in ((-1, 4, 1), (1, 0, 1), (1, 4, 0), (2 ** 31, 4, 1),
                             (1, 2 ** 30 + 1, 1)):
    assert lib.xse_mxfp4_codes_bytes(rows, cols, groups) == 0
    assert lib.xse_mxfp4_scales_bytes(rows, cols, groups) == 0
  assert lib.xse_expert_linear_workspace(8, 0, 64) == 0
  assert lib.xse_expert_linear_workspace(8, 1025, 64) == 0
  assert lib.xse_expert_linear_workspace(8, 4, 64) == 0
  assert lib.xse_expert_linear_workspace(800, 4, 64) >= 800 * 32 + 7 * 512


def test_expert_scale_tiles_never_overlap():
  """The closed form of an expert's first scale tile (offsets[e] / n + e)
  leaves each expert its tiles, and the last ends within pairs / n + experts."""
  rng = np.random.default_rng(0)
  for n in (16, 32, 64, 128):
    for _ in range(300):
      experts = int(rng.integers(1, 40))
      counts = rng.integers(0, 3 * n, experts) * (rng.random(experts) < 0.7)
      offsets = np.concatenate([[0], np.cumsum(counts)])
      pairs = int(offsets[-1] + rng.integers(0, 5))
      first = offsets[:-1] // n + np.arange(experts)
      last = first + -(-counts // n)
      assert (last[:-1] <= first[1:]).all()
      assert last[-1] <= pairs // n + experts


def test_expert_scale_tiles_of_pairs_never_overlap(capi):
  """Tiles of 256 rows take two scale tiles of 128 rows each: an expert's rows
  still have scale tiles of their own, and the workspace holds the last."""
  rng = np.random.default_rng(2)
  n, cols = 256, 1536
  for _ in range(300):
    experts = int(rng.integers(1, 40))
    counts = rng.integers(0, 3 * n, experts) * (rng.random(experts) < 0.7)
    offsets = np.concatenate([[0], np.cumsum(counts)])
    pairs = int(offsets[-1] + rng.integers(0, 5))
    first = (offsets[:-1] // n + np.arange(experts)) * 2
    last = first + -(-counts // 128)
    assert (last[:-1] <= first[1:]).all()
    assert last[-1] <= (pairs // n + experts) * 2
    if pairs > 128 * experts:  # the rule for such tiles
      need = capi.lib.xse_expert_linear_workspace(pairs, experts, cols)
      assert need >= pairs * cols // 2 + last[-1] * (cols // 128) * 512


def test_reference_quantisation_by_search():
  """The reference's codes are a nearest grid value to the scaled element, the
  even one at a tie."""
  rng = np.random.default_rng(1)
  x = np.concatenate([rng.standard_normal((8, 64)),
                      rng.integers(-32, 33, (8, 64)) / 4.0])
  codes, s = ref.quantize(x)
  scaled = np.abs(x) / np.repeat(np.exp2(s - 127.0), 32, axis=1)
  gap = np.abs(scaled[..., None] - ref.GRID)
  best = gap.min(-1)
  mine = codes & 7
  assert (np.take_along_axis(gap, mine[..., None], -1)[..., 0] == best).all()
  tied = (gap == best[..., None]).sum(-1) > 1
  assert tied.any() and (mine[tied] % 2 == 0).all()
  np.testing.assert_array_equal(np.signbit(x), (codes & 8) != 0)


def test_matrix_refusals(capi):
  lib = capi.lib
  q = lambda m, dtype=0: lib.xse_mxfp4_quantize(4096, dtype, 0, 64, 1, m, None)  # noqa: E731
  refused(capi, q(None), "4-bit matrix q")
  refused(capi, q(matrix(capi, rows=-1)), "rows")
  refused(capi, q(matrix(capi, rows=2 ** 31)), "rows")
  refused(capi, q(matrix(capi, cols=0)), "cols")
  refused(capi, q(matrix(capi, cols=2 ** 30 + 1)), "cols")
  refused(capi, q(matrix(capi, groups=0)), "groups")
  refused(capi, q(matrix(capi, codes=None)), "non-null")
  refused(capi, q(matrix(capi, codes=4104)), "aligned")
  refused(capi, q(matrix(capi, scales=8)), "aligned")
  refused(capi, q(matrix(capi), dtype=2), "type 2")
  refused(capi, lib.xse_mxfp4_quantize(None, 0, 0, 64, 1, matrix(capi), None),
          "null")
  d = lambda m, out=4096, dtype=0, stride=64: lib.xse_mxfp4_dequantize(  # noqa: E731
      m, out, dtype, 0, stride, None)
  refused(capi, d(matrix(capi), stride=63), "stride")
  refused(capi, d(matrix(capi), dtype=7), "type 7")
  refused(capi, d(matrix(capi), out=None), "null")
  assert q(matrix(capi, rows=0, codes=None, scales=None)) == capi.OK
  assert d(matrix(capi, rows=0, codes=None, scales=None)) == capi.OK


@pytest.mark.parametrize("rows,cols,groups", [
    (2 ** 30, 512, 2 ** 30),        # both sizes a multiple of 2^64
    (2 ** 30, 2 ** 29, 1024),
    (2 ** 30, 32, 2 ** 30), (2 ** 31 - 1, 2 ** 30, 2 ** 31 - 1),
    (2 ** 31 - 1, 2 ** 30, 9)])
def test_matrices_past_63_bits(capi, xse, rows, cols, groups):
  """Their bytes have no number: nobody can have allocated them."""
  lib = capi.lib
  assert groups * rows * -(-cols // 32) * 16 >= 2 ** 63
  assert lib.xse_mxfp4_codes_bytes(rows, cols, groups) == 0
  assert lib.xse_mxfp4_scales_bytes(rows, cols, groups) == 0
  q = matrix(capi, rows, cols, groups)
  refused(capi, lib.xse_mxfp4_quantize(4096, 0, 0, 0, 0, q, None), "2^63")
  refused(capi, lib.xse_mxfp4_dequantize(q, 4096, 0, 0, cols, None), "2^63")
  buffer = types.SimpleNamespace(
      dtype=torch.uint8, is_contiguous=lambda: True, is_cuda=True,
      numel=lambda: 4096, device="cuda:0", data_ptr=lambda: 4096,
      get_device=lambda: 0)
  with pytest.raises(xse.XseError, match="2.63"):
    xse.mx.MxMatrix(buffer, buffer, rows, cols, groups)


def test_the_largest_sizes(capi):
  rows, cols = 2 ** 31 - 1, 2 ** 30
  assert capi.lib.xse_mxfp4_codes_bytes(rows, cols, 7) == 7 * rows * 2 ** 29
  assert capi.lib.xse_mxfp4_scales_bytes(rows, cols, 7) == \
      7 * 2 ** 24 * 2 ** 23 * 512


def test_layer_refusals(capi):
  lib = capi.lib

  def layer(x=4096, dtype=0, rows=40, stride=64, w=None, act=0, y=4096,
            y_type=0, y_stride=32, scratch=4096, size=1 << 20):
    return lib.xse_linear_forward_mxfp4(
        x, dtype, rows, stride, w or matrix(capi, rows=32), None, act, y,
        y_type, y_stride, scratch, size, None)

  refused(capi, layer(dtype=2), "type 2")
  refused(capi, layer(rows=-1), "rows")
  refused(capi, layer(stride=63), "stride")
  refused(capi, layer(w=matrix(capi, rows=0)), "output row")
  refused(capi, layer(w=matrix(capi, rows=32, groups=2)), "one group")
  refused(capi, layer(act=3), "activation")
  refused(capi, layer(y_type=2), "type 2")
  refused(capi, layer(y_stride=31), "stride")
  refused(capi, layer(x=None), "non-null")
  refused(capi, layer(y=None), "non-null")
  refused(capi, layer(scratch=None), "non-null")
  refused(capi, layer(scratch=4100), "aligned")
  refused(capi, layer(size=lib.xse_linear_mxfp4_workspace(40, 64) - 1),
          "workspace")
  assert layer(rows=0, x=None, y=None, scratch=None, size=0) == capi.OK
  two = lib.xse_linear_forward_mxfp4_q
  refused(capi, two(matrix(capi, cols=32), matrix(capi, rows=32), None, 0,
                    4096, 0, 32, None), "columns")
  refused(capi, two(matrix(capi, groups=2), matrix(capi, rows=32), None, 0,
                    4096, 0, 32, None), "one group")


def test_expert_refusals(capi):
  lib = capi.lib
  sort = lambda p, kind=0, ids=4096, w=None, n=0: lib.xse_expert_sort(  # noqa: E731
      ids, kind, p, w, n, None)
  refused(capi, sort(None), "plan")
  refused(capi, sort(plan(capi, tokens=-1)), "tokens")
  refused(capi, sort(plan(capi, topk=0)), "topk")
  refused(capi, sort(plan(capi, experts=0)), "experts")
  refused(capi, sort(plan(capi, experts=1025)), "experts")
  refused(capi, sort(plan(capi, tokens=2 ** 30, topk=2)), "2^31")
  refused(capi, sort(plan(capi, offsets=None)), "non-null")
  refused(capi, sort(plan(capi, slots=None)), "non-null")
  refused(capi, sort(plan(capi), kind=2), "int32 or int64")
  refused(capi, sort(plan(capi), ids=None), "non-null")
  need = lib.xse_expert_sort_workspace(100000, 3)
  assert need > 0 and lib.xse_expert_sort_workspace(8, 3) == 0
  large = plan(capi, tokens=50000)
  refused(capi, sort(large), "workspace")
  refused(capi, sort(large, w=4096, n=need - 1), "workspace")
  refused(capi, sort(large, w=4098, n=need), "aligned")

  def gather(p=None, dtype=0, cols=64, x=4096, xs=64, out=4096, os=64):
    return lib.xse_expert_gather(x, dtype, cols, xs, p or plan(capi), out, os,
                                 None)

  def combine(p=None, dtype=0, cols=64, y=4096, ys=64, out=4096, os=64):
    return lib.xse_expert_combine(y, dtype, cols, ys, p or plan(capi), None,
                                  out, os, None)

  for call, first in ((gather, "x"), (combine, "y")):
    refused(capi, call(dtype=2), "type 2")
    refused(capi, call(cols=0), "cols")
    refused(capi, call(cols=2 ** 30 + 1, os=2 ** 31, **{first + "s": 2 ** 31}),
            "cols")
    refused(capi, call(os=63), "strides")
    refused(capi, call(**{first + "s": 63}), "strides")
    refused(capi, call(**{first: None}), "non-null")
    refused(capi, call(out=None), "non-null")
    empty = plan(capi, tokens=0, order=None, slots=None)
    assert call(p=empty, out=None, **{first: None}) == capi.OK

  def backward(grad=4096, y=4096, ys=64, gy=4096, gys=64, gw=4096):
    return lib.xse_expert_combine_backward(grad, y, 0, 64, 64, ys, plan(capi),
                                           None, gy, gys, gw, None)

  refused(capi, backward(grad=None), "non-null")
  refused(capi, backward(y=None), "non-null")
  refused(capi, backward(ys=63), "strides")
  refused(capi, backward(gys=63), "strides")
  assert backward(gy=None, gw=None) == capi.OK

  def layer(groups=3, size=1 << 20, flag=0, stride=64):
    return lib.xse_expert_linear_mxfp4(
        4096, 0, stride, flag, plan(capi, tokens=400),
        matrix(capi, rows=32, groups=groups),
        None, 0, 4096, 0, 32, 4096, size, None)

  refused(capi, layer(groups=2), "one group of w per expert")
  refused(capi, layer(size=0), "workspace")
  refused(capi, layer(stride=1, flag=1), "stride")
