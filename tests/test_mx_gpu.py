"""Microscaled 4-bit matrices and layers (include/xse_mx.h) against 64-bit
references. Quantisation is exact up to its one rounding, whose rule the
reference restates, so codes and scales are compared bit for bit; a layer's
tolerance is derived in mx_reference.linear_tolerance."""

import numpy as np
import pytest
import torch

from tests import mx_reference as ref

pytestmark = pytest.mark.gpu

EPS = {torch.float32: 2.0 ** -23, torch.bfloat16: 2.0 ** -7}


@pytest.fixture(scope="module")
def mx(xse):
  return xse.mx


def make(rows, cols, dtype, seed=0, scale=True):
  gen = torch.Generator().manual_seed(seed * 7919 + rows * 31 + cols)
  x = torch.randn((rows, cols), generator=gen)
  if scale:
    x *= torch.exp2(torch.randint(-12, 12, (rows, 1), generator=gen).float())
  return x.to(dtype)


def check_quantized(q, x, group=0):
  """Codes and scales of one group against the reference's."""
  rows, cols = x.shape
  codes, s = ref.quantize(x.double().numpy())
  row_bytes = 16 * -(-cols // 32)
  per = rows * row_bytes
  got = q.codes.cpu().numpy()[group * per:(group + 1) * per]
  np.testing.assert_array_equal(got.reshape(rows, row_bytes),
                                ref.pack_codes(codes))
  tiles = -(-rows // 128) * -(-cols // 128) * 512
  got = q.scales.cpu().numpy()[group * tiles:(group + 1) * tiles]
  blocks = s.shape[1]
  padded = -(-blocks // 4) * 4
  want = np.zeros((rows, padded), np.int64)  # pad blocks of a tile are 0
  want[:, :blocks] = s
  np.testing.assert_array_equal(got[ref.scale_offsets(rows, padded)], want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [
    (1, 1), (1, 32), (3, 13), (2, 33), (5, 128), (129, 160), (7, 479),
    (260, 256), (33, 1000), (4, 4096)])
def test_quantize(mx, dtype, rows, cols):
  x = make(rows, cols, dtype)
  q = mx.quantize(x.cuda())
  check_quantized(q, x)
  want = ref.quantized(x.double().numpy())
  for out_type in (torch.float32, torch.bfloat16):
    got = mx.dequantize(q, dtype=out_type)
    assert got.dtype == out_type
    np.testing.assert_array_equal(got.double().cpu().numpy(), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize_strides(mx, dtype):
  base = make(70, 400, dtype, seed=1)
  dev = base.cuda()
  for view, host in (
      (dev[:, 3:260], base[:, 3:260]),      # unaligned rows
      (dev[1:, 8:264], base[1:, 8:264]),    # aligned, padded rows
      (dev.t(), base.t()),                  # rows along the last axis
      (dev[::2, ::3], base[::2, ::3]),      # both apart
      (dev[4:5].expand(5, -1), base[4:5].expand(5, -1))):
    q = mx.quantize(view)
    check_quantized(q, host)
    np.testing.assert_array_equal(
        mx.dequantize(q).double().cpu().numpy(),
        ref.quantized(host.double().numpy()))


@pytest.mark.parametrize("shape,transposed", [
    ((3, 50, 96), False), ((2, 130, 77), False), ((4, 64, 200), True)])
def test_quantize_groups(mx, shape, transposed):
  gen = torch.Generator().manual_seed(sum(shape))
  x = torch.randn(shape, generator=gen)
  view = x.cuda()
  if transposed:
    x, view = x.transpose(1, 2), view.transpose(1, 2)
  q = mx.quantize(view)
  for g in range(shape[0]):
    check_quantized(q, x[g], g)
  got = mx.dequantize(q).double().cpu().numpy()
  for g in range(shape[0]):
    np.testing.assert_array_equal(got[g], ref.quantized(x[g].double().numpy()))


def special_blocks():
  blocks = []
  ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.9])
  blocks.append(torch.cat([ties, -ties, torch.zeros(12)]))
  blocks.append(torch.zeros(32))
  blocks.append(-torch.zeros(32))
  blocks.append(torch.full((32,), 2.0 ** -149))           # subnormal
  blocks.append(torch.linspace(0, 2.0 ** -126, 32))       # around the smallest
  blocks.append(torch.linspace(-3.0e38, 3.4e38, 32))      # around the largest
  for k in (-149, -140, -127, -126, -125, -124, -3, 0, 1, 2, 3, 126, 127):
    b = torch.zeros(32)
    b[5] = 2.0 ** k                                       # powers of two
    b[6] = -0.5 * 2.0 ** k
    blocks.append(b)
    blocks.append(b * (1 - 2.0 ** -24) if k > -126 else b)
  for v in (float("inf"), -float("inf"), float("nan")):
    b = torch.linspace(-1, 1, 32)
    b[17] = v
    blocks.append(b)
  return torch.stack(blocks)


@pytest.mark.parametrize("offset", [0, 1])
def test_quantize_special(mx, offset):
  x = special_blocks()
  # One block a row, and all blocks in one row (a bad block spoils no other),
  # through the aligned kernel and the unaligned one.
  for host in (x, x.reshape(1, -1)):
    buf = torch.zeros((host.shape[0], host.shape[1] + 8))
    buf[:, offset:offset + host.shape[1]] = host
    view = buf.cuda()[:, offset:offset + host.shape[1]]
    q = mx.quantize(view)
    check_quantized(q, host)
    want = ref.quantized(host.double().numpy())
    np.testing.assert_array_equal(
        mx.dequantize(q).double().cpu().numpy(), want)
    np.testing.assert_array_equal(
        mx.dequantize(q, dtype=torch.bfloat16).double().cpu().numpy(), want)
    check_quantized(mx.quantize(view.t().contiguous().t()), host)


def test_dequantize_leaves_the_rest(mx):
  x = make(9, 45, torch.float32)
  q = mx.quantize(x.cuda())
  buf = torch.full((12, 64), 7.0, device="cuda")
  mx.dequantize(q, buf[1:10, 3:48])
  got = buf.cpu()
  np.testing.assert_array_equal(got[1:10, 3:48].double().numpy(),
                                ref.quantized(x.double().numpy()))
  got[1:10, 3:48] = 7.0
  assert bool((got == 7.0).all())


def weights(mx, out, cols, seed=0):
  """(MxMatrix, its values in 64 bits) of a random [out, cols]."""
  w = make(out, cols, torch.float32, seed + 100, scale=False) * cols ** -0.5
  return mx.quantize(w.cuda()), ref.quantized(w.double().numpy())


LAYERS = [  # rows, in, out
    (1, 1, 1), (1, 32, 128), (3, 64, 7), (16, 256, 130), (17, 257, 128),
    (5, 13, 512), (33, 100, 64), (64, 320, 200), (65, 128, 129),
    (100, 479, 1024), (128, 512, 256), (300, 96, 333), (1, 4096, 1024),
    (20, 3000, 140), (700, 600, 512), (2, 2048, 4096), (257, 1536, 128),
    (700, 1700, 390), (129, 2048, 7), (513, 2100, 1000), (40, 9000, 130),
    (8, 9000, 33)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols,out", LAYERS)
def test_linear(mx, rows, cols, out, dtype):
  x = make(rows, cols, dtype, seed=2, scale=rows % 2 == 0)
  w, w_values = weights(mx, out, cols)
  gen = torch.Generator().manual_seed(out)
  bias = torch.randn((out,), generator=gen)
  for b, act in ((None, 0), (bias, 1), (bias, 2)):
    y = mx.linear(x.cuda(), w, None if b is None else b.cuda(), act)
    assert y.dtype == dtype and y.shape == (rows, out)
    want, size = ref.linear(x.double().numpy(), w_values,
                            None if b is None else b.double().numpy(), act)
    np.testing.assert_array_less(
        np.abs(y.double().cpu().numpy() - want),
        ref.linear_tolerance(want, size, cols, EPS[dtype]))
  mx.check()


@pytest.mark.parametrize("rows", [4, 150])
def test_linear_strides_and_types(mx, rows):
  """Strided x and y, the other output type, x quantised before: all give the
  numbers of the plain call, and nothing outside y is written."""
  cols, out = 333, 150
  x = make(rows, cols, torch.float32, seed=3)
  w, _ = weights(mx, out, cols)
  plain = mx.linear(x.cuda(), w)
  buf = torch.zeros((rows, cols + 9), device="cuda")
  buf[:, 5:5 + cols] = x.cuda()
  y = torch.full((rows + 2, out + 6), 7.0, device="cuda")
  mx.linear(buf[:, 5:5 + cols], w, out=y[1:-1, 3:-3])
  assert torch.equal(y[1:-1, 3:-3], plain)
  y[1:-1, 3:-3] = 7.0
  assert bool((y == 7.0).all())
  assert torch.equal(mx.linear(mx.quantize(x.cuda()), w), plain)
  half = torch.empty((rows, out), dtype=torch.bfloat16, device="cuda")
  mx.linear(x.cuda(), w, out=half)
  assert torch.equal(half, plain.bfloat16())


@pytest.mark.parametrize("rows", [6, 200])
def test_linear_nan_stays_in_its_row(mx, rows):
  cols, out = 200, 140
  x = make(rows, cols, torch.float32, seed=4)
  w, w_values = weights(mx, out, cols)
  x[2, 50] = float("inf")
  x[4, 199] = float("nan")
  y = mx.linear(x.cuda(), w, None, mx.ACT_RELU).double().cpu().numpy()
  bad = np.zeros(rows, bool)
  bad[[2, 4]] = True
  assert np.isnan(y[bad]).all()
  want, size = ref.linear(x.double().numpy()[~bad], w_values, None, 1)
  np.testing.assert_array_less(
      np.abs(y[~bad] - want),
      ref.linear_tolerance(want, size, cols, EPS[torch.float32]))


def test_linear_repeats_bit_for_bit(mx):
  for rows, cols, out in ((3, 4096, 256), (513, 1024, 384)):
    x = make(rows, cols, torch.bfloat16, seed=5).cuda()
    w, _ = weights(mx, out, cols)
    first = mx.linear(x, w)
    for _ in range(5):
      assert torch.equal(mx.linear(x, w), first)


# rows, in, out: three tiles or more for every block, in each form of the
# product (tiles of 16, 32, 64 and 128 rows, pairs of blocks with an even and an
# odd number of feature tiles).
MANY_TILES = [
    (10, 500, 60_000), (30, 500, 60_001), (60, 700, 60_000), (2100, 300, 4000),
    (2100, 1600, 6400), (2100, 1600, 6500)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols,out", MANY_TILES)
def test_linear_of_many_tiles(mx, rows, cols, out, dtype):
  """Against 64 bits (summed on the device: some 40 GFLOP)."""
  x = make(rows, cols, dtype, seed=9)
  w, w_values = weights(mx, out, cols)
  gen = torch.Generator().manual_seed(out)
  bias = torch.randn((out,), generator=gen)
  y = mx.linear(x.cuda(), w, bias.cuda(), mx.ACT_RELU)
  q = torch.from_numpy(ref.quantized(x.double().numpy())).cuda()
  v, b = torch.from_numpy(w_values).cuda(), bias.double().cuda()
  want = torch.relu(q @ v.t() + b)
  size = q.abs() @ v.abs().t() + b.abs()
  bound = (ref.linear_tolerance(0.0, size, cols, EPS[dtype]) +
           EPS[dtype] / 2 * want)
  assert bool(((y.double() - want).abs() <= bound).all())
  again = mx.linear(x.cuda(), w, bias.cuda(), mx.ACT_RELU)
  assert torch.equal(again, y)
  mx.check()


PAIRS = (300, 2048, 390)  # rows, in, out of a product by pairs of blocks


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_pairs_strides_and_types(mx, dtype):
  """Strided x and y (rows of y an even and an odd number of elements apart and
  at odd offsets), the other output type, x quantised before: the numbers of
  the plain call, and nothing outside y is written."""
  rows, cols, out = PAIRS
  x = make(rows, cols, dtype, seed=10)
  w, _ = weights(mx, out, cols)
  plain = mx.linear(x.cuda(), w)
  exact = mx.linear(x.cuda(), w, out=torch.empty((rows, out), device="cuda"))
  assert torch.equal(exact.to(dtype), plain)
  buf = torch.zeros((rows, cols + 9), dtype=dtype, device="cuda")
  buf[:, 5:5 + cols] = x.cuda()
  for left, right in ((2, 4), (3, 3), (3, 4)):
    y = torch.full((rows + 2, left + out + right), 7.0, dtype=dtype,
                   device="cuda")
    view = y[1:-1, left:left + out]
    mx.linear(buf[:, 5:5 + cols], w, out=view)
    assert torch.equal(view, plain)
    view.fill_(7.0)
    assert bool((y == 7.0).all())
  q = mx.quantize(x.cuda())
  assert torch.equal(mx.linear(q, w), exact)
  half = torch.empty((rows, out), dtype=torch.bfloat16, device="cuda")
  assert torch.equal(mx.linear(q, w, out=half), exact.bfloat16())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_pairs_keep_nan_in_its_row(mx, dtype):
  rows, cols, out = PAIRS
  x = make(rows, cols, dtype, seed=11)
  w, w_values = weights(mx, out, cols)
  bad = np.zeros(rows, bool)
  for row, col, value in ((0, 0, "nan"), (127, 2047, "inf"), (128, 1024, "-inf"),
                          (255, 31, "nan"), (256, 32, "inf"), (299, 5, "nan")):
    x[row, col] = float(value)
    bad[row] = True
  y = mx.linear(x.cuda(), w, None, mx.ACT_RELU).double().cpu().numpy()
  assert np.isnan(y[bad]).all()
  want, size = ref.linear(x.double().numpy()[~bad], w_values, None, 1)
  bound = ref.linear_tolerance(want, size, cols, EPS[dtype])
  assert (np.abs(y[~bad] - want) <= bound).all()


def test_pairs_on_other_streams_and_in_graphs(mx):
  """Repeats, two streams at once, and two graphs replayed together."""
  rows, cols, out = PAIRS
  w, _ = weights(mx, out, cols)
  xs = [make(n, cols, torch.bfloat16, seed=12 + n).cuda()
        for n in (rows, 2000)]
  want = [mx.linear(x, w) for x in xs]
  torch.cuda.synchronize()
  streams = [torch.cuda.Stream() for _ in xs]
  for _ in range(20):
    got = [mx.linear(x, w, stream=s) for x, s in zip(xs, streams)]
    torch.cuda.synchronize()
    for a, b in zip(got, want):
      assert torch.equal(a, b)
  graphs, outs = [], []
  for x in xs:
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
      outs.append(mx.linear(x, w))
    graphs.append(g)
  for _ in range(5):
    for o in outs:
      o.zero_()
    torch.cuda.synchronize()
    for g, s in zip(graphs, streams):
      with torch.cuda.stream(s):
        g.replay()
    torch.cuda.synchronize()
    for a, b in zip(outs, want):
      assert torch.equal(a, b)
  mx.check()


def test_linear_empty(mx):
  w, _ = weights(mx, 64, 96)
  y = mx.linear(torch.zeros((0, 96), device="cuda"), w)
  assert y.shape == (0, 64)
  q = mx.quantize(torch.zeros((0, 96), device="cuda"))
  assert mx.dequantize(q).shape == (0, 96)
  assert mx.linear(q, w).shape == (0, 64)


def test_linear_on_other_streams_and_in_graphs(mx):
  """Concurrent calls on two streams, and two graphs of the same layer
  replayed in turn and together, each with its own scratch."""
  w, _ = weights(mx, 256, 512)
  xs = [make(rows, 512, torch.float32, seed=6 + rows).cuda()
        for rows in (4, 300)]
  want = [mx.linear(x, w) for x in xs]
  torch.cuda.synchronize()
  streams = [torch.cuda.Stream() for _ in xs]
  for _ in range(20):
    got = [mx.linear(x, w, stream=s) for x, s in zip(xs, streams)]
    torch.cuda.synchronize()
    for a, b in zip(got, want):
      assert torch.equal(a, b)
  graphs, outs = [], []
  for x in xs:
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
      outs.append(mx.linear(x, w))
    graphs.append(g)
  for _ in range(5):
    for o in outs:
      o.zero_()
    torch.cuda.synchronize()
    for g, s in zip(graphs, streams):
      with torch.cuda.stream(s):
        g.replay()
    torch.cuda.synchronize()
    for a, b in zip(outs, want):
      assert torch.equal(a, b)


def test_offsets_past_32_bits(mx):
  """More than 2^32 elements in x and in y."""
  rows, cols = 70_000, 65_536
  x = torch.empty((rows, cols), dtype=torch.bfloat16, device="cuda")
  for part in x.split(10_000):
    part.normal_()
  q = mx.quantize(x)
  back = mx.dequantize(q, dtype=torch.bfloat16)
  for r in (0, 65_537, rows - 1):
    np.testing.assert_array_equal(
        back[r:r + 1].double().cpu().numpy(),
        ref.quantized(x[r:r + 1].double().cpu().numpy()))
  del x, q, back
  w, _ = weights(mx, 32, 64)
  x = make(40_000, 64, torch.float32, seed=8).cuda()
  y = torch.empty((40_000, 110_000), device="cuda")[:, :32]
  mx.linear(x, w, out=y)
  assert torch.equal(y, mx.linear(x, w))


def test_row_whose_scales_pass_32_bits(mx):
  """A row of more than 2^29 columns: its scale tiles take more than 2^31
  bytes. Blocks do not depend on one another, so shorter rows give its values."""
  cols, short = 2 ** 29 + 4096, 4096
  x = torch.empty((1, cols), dtype=torch.bfloat16, device="cuda")
  gen = torch.Generator(device="cuda").manual_seed(0)
  for part in x.view(-1).split(2 ** 26):
    part.normal_(generator=gen)
  want = mx.dequantize(mx.quantize(x.view(-1, short)), dtype=x.dtype)
  q = mx.quantize(x)
  assert q.scales.numel() > 2 ** 31
  got = mx.dequantize(q, dtype=x.dtype)
  assert torch.equal(got.view(-1, short), want)
  np.testing.assert_array_equal(
      got[:, -short:].double().cpu().numpy(),
      ref.quantized(x[:, -short:].double().cpu().numpy()))
  odd = torch.empty((1, cols + 1), device="cuda")[:, 1:]  # off the 16-byte grid
  mx.dequantize(q, odd)
  assert torch.equal(odd, got.float())


def test_refusals(mx, xse):
  x = torch.zeros((4, 64), device="cuda")
  w, _ = weights(mx, 32, 64)
  cases = [
      lambda: mx.quantize(x.half()),
      lambda: mx.quantize(x.cpu()),
      lambda: mx.quantize(x[0]),
      lambda: mx.quantize(x, mx.MxMatrix.empty(4, 96)),
      lambda: mx.dequantize(mx.quantize(x), torch.zeros((4, 65),
                                                        device="cuda")),
      lambda: mx.dequantize(mx.quantize(x), dtype=torch.float16),
      lambda: mx.linear(x[:, :32], w),
      lambda: mx.linear(x.t(), w),
      lambda: mx.linear(x, w, torch.zeros(31, device="cuda")),
      lambda: mx.linear(x, w, torch.zeros(32, device="cuda").bfloat16()),
      lambda: mx.linear(x, w, None, 9),
      lambda: mx.linear(x, w, out=torch.zeros((4, 31), device="cuda")),
      lambda: mx.linear(x, w, out=torch.zeros((32, 4), device="cuda").t()),
      lambda: mx.linear(x.cpu(), w),
      lambda: mx.linear(x, mx.quantize(torch.zeros((2, 32, 64),
                                                   device="cuda"))),
      lambda: mx.linear(mx.quantize(x[:, :32]), w),
  ]
  for case in cases:
    with pytest.raises(xse.XseError) as e:
      case()
    assert e.value.code == xse._capi.INVALID_ARGUMENT
