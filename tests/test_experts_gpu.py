"""Rows sorted by expert and back, and the experts' 4-bit layers
(include/xse_experts.h) against 64-bit references.

Tolerances. gather moves rows unchanged. combine adds topk products in fp32:
each product and addition is off by at most half a unit (2^-24) of the sum of
magnitudes so far, so the sum by at most 2 topk 2^-24 of it, and one rounding
to the output's type by eps / 2. A weight's gradient adds cols products: 2 cols
2^-24 of the sum of magnitudes. The layers as in mx_reference."""

import numpy as np
import pytest
import torch

from tests import mx_reference as ref

pytestmark = pytest.mark.gpu

EPS = {torch.float32: 2.0 ** -23, torch.bfloat16: 2.0 ** -7}


@pytest.fixture(scope="module")
def mx(xse):
  return xse.mx


@pytest.fixture(scope="module")
def experts(xse):
  return xse.experts


def choose(tokens, topk, num_experts, seed=0, dropped=0.1, skew=True):
  """Expert ids with some pairs dropped, a token of none, one expert twice."""
  rng = np.random.default_rng(seed + tokens * 131 + topk * 17 + num_experts)
  p = rng.dirichlet(np.full(num_experts, 0.5 if skew else 50.0))
  ids = rng.choice(num_experts, (tokens, topk), p=p).astype(np.int64)
  ids[rng.random((tokens, topk)) < dropped] = -1
  if tokens > 3:
    ids[tokens // 2] = -1
    ids[1] = num_experts - 1
    ids[2, 0] = num_experts  # out of range, dropped
  return ids


PLANS = [  # tokens, topk, experts
    (1, 1, 1), (1, 8, 64), (5, 2, 3), (64, 4, 64), (100, 8, 128),
    (333, 3, 1024), (1025, 4, 7), (4096, 2, 256), (20000, 8, 130),
    (70001, 1, 33)]


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("tokens,topk,num_experts", PLANS)
def test_sort(experts, tokens, topk, num_experts, dtype):
  ids = choose(tokens, topk, num_experts)
  plan = experts.sort(torch.from_numpy(ids).to(dtype).cuda(), num_experts)
  offsets, order, slots = ref.sort(ids, num_experts)
  np.testing.assert_array_equal(plan.offsets.cpu().numpy(), offsets)
  np.testing.assert_array_equal(plan.order.cpu().numpy(), order)
  np.testing.assert_array_equal(plan.slots.cpu().numpy(), slots)


def test_sort_extremes(experts):
  for ids, num_experts in (
      (np.full((5000, 2), -1), 16),                 # nothing kept
      (np.full((5000, 2), 15), 16),                 # all in one expert
      (np.full((300, 1), 2 ** 40), 4),              # far out of range
      (np.full((300, 1), -2 ** 40 + 1), 4),
      (np.arange(8192).reshape(-1, 2) % 1024, 1024)):
    plan = experts.sort(torch.from_numpy(ids).cuda(), num_experts)
    for got, want in zip((plan.offsets, plan.order, plan.slots),
                         ref.sort(ids, num_experts)):
      np.testing.assert_array_equal(got.cpu().numpy(), want)
  plan = experts.sort(torch.zeros((0, 4), dtype=torch.int32, device="cuda"), 9)
  assert plan.offsets.tolist() == [0] * 10 and plan.slots.shape == (0, 4)


def make(rows, cols, dtype, seed):
  gen = torch.Generator().manual_seed(seed * 7919 + rows * 31 + cols)
  return torch.randn((rows, cols), generator=gen).to(dtype)


ROWS = [  # tokens, topk, experts, cols
    (1, 1, 1, 1), (3, 2, 4, 7), (64, 4, 64, 256), (50, 3, 5, 479),
    (129, 8, 16, 1032), (1000, 2, 8, 64), (17, 6, 3, 4096),
    (20, 12, 30, 136), (9, 40, 50, 77), (3, 40, 64, 128)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens,topk,num_experts,cols", ROWS)
def test_gather_and_combine(experts, tokens, topk, num_experts, cols, dtype):
  ids = choose(tokens, topk, num_experts, seed=1)
  plan = experts.sort(torch.from_numpy(ids).cuda(), num_experts)
  _, order, slots = ref.sort(ids, num_experts)
  x = make(tokens, cols, dtype, 1)
  got = experts.gather(x.cuda(), plan)
  want = np.where(order[:, None] >= 0, x.double().numpy()[order // topk], 0.0)
  assert got.dtype == dtype
  np.testing.assert_array_equal(got.double().cpu().numpy(), want)

  y = make(tokens * topk, cols, dtype, 2)
  y[(order < 0).nonzero()[0]] = float("nan")  # rows behind the last: not read
  w = make(tokens, topk, torch.float32, 3)
  kept = (slots >= 0)[..., None]
  rows = np.where(kept, y.double().numpy()[slots], 0.0)
  for weights in (w, None):
    got = experts.combine(y.cuda(), plan,
                          None if weights is None else weights.cuda())
    f = 1.0 if weights is None else weights.double().numpy()[..., None]
    want, size = (f * rows).sum(1), np.abs(f * rows).sum(1)
    assert got.dtype == dtype
    bound = 2 * topk * 2.0 ** -24 * size + EPS[dtype] / 2 * np.abs(want)
    assert (np.abs(got.double().cpu().numpy() - want) <= bound).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens,topk,num_experts,cols", ROWS)
def test_combine_backward(experts, tokens, topk, num_experts, cols, dtype):
  ids = choose(tokens, topk, num_experts, seed=2)
  plan = experts.sort(torch.from_numpy(ids).cuda(), num_experts)
  _, order, slots = ref.sort(ids, num_experts)
  y, grad = make(tokens * topk, cols, dtype, 4), make(tokens, cols, dtype, 5)
  y[(order < 0).nonzero()[0]] = float("nan")
  w = make(tokens, topk, torch.float32, 6)
  gy, gw = experts.combine_backward(grad.cuda(), y.cuda(), plan, w.cuda())
  g = grad.double().numpy()
  want = np.where(order[:, None] >= 0,
                  w.double().numpy().reshape(-1)[order][:, None] *
                  g[order // topk], 0.0)
  assert gy.dtype == dtype and gw.dtype == torch.float32
  assert (np.abs(gy.double().cpu().numpy() - want) <=
          (EPS[dtype] / 2 + 2.0 ** -24) * np.abs(want)).all()
  kept = (slots >= 0)[..., None]
  parts = np.where(kept, y.double().numpy()[slots], 0.0) * g[:, None, :]
  assert (np.abs(gw.double().cpu().numpy() - parts.sum(2)) <=
          2 * cols * 2.0 ** -24 * np.abs(parts).sum(2)).all()
  one, _ = experts.combine_backward(grad.cuda(), y.cuda(), plan)
  assert torch.equal(one, experts.gather(grad.cuda(), plan))


def test_gradients_against_differences(experts):
  """combine is linear in y and in the weights, and gather in x: a step's
  difference is the gradient's product with it, up to the roundings of three
  fp32 sums."""
  tokens, topk, num_experts, cols = 40, 4, 6, 96
  ids = choose(tokens, topk, num_experts, seed=3)
  plan = experts.sort(torch.from_numpy(ids).cuda(), num_experts)
  y, dy = (make(tokens * topk, cols, torch.float32, s).cuda() for s in (7, 8))
  w, dw = (make(tokens, topk, torch.float32, s).cuda() for s in (9, 10))
  grad = make(tokens, cols, torch.float32, 11).cuda()
  gy, gw = experts.combine_backward(grad, y, plan, w)
  dot = lambda a, b: (a.double() * b.double()).sum().item()  # noqa: E731
  base = experts.combine(y, plan, w)
  for stepped, want in ((experts.combine(y + dy, plan, w), dot(gy, dy)),
                        (experts.combine(y, plan, w + dw), dot(gw, dw))):
    got = dot(grad, stepped) - dot(grad, base)
    size = dot(grad.abs(), stepped.abs()) + dot(grad.abs(), base.abs())
    assert abs(got - want) <= 16 * 2.0 ** -24 * cols * size
  x, dx = (make(tokens, cols, torch.float32, s).cuda() for s in (12, 13))
  gs = make(tokens * topk, cols, torch.float32, 14).cuda()
  got = dot(gs, experts.gather(x + dx, plan)) - dot(gs, experts.gather(x, plan))
  want = dot(experts.combine(gs, plan), dx)
  size = dot(gs.abs(), experts.gather(x.abs() + dx.abs(), plan))
  assert abs(got - want) <= 16 * 2.0 ** -24 * size


def test_strided_rows(experts):
  """Rows in wider buffers, at offsets that rule out whole vectors; nothing
  outside the outputs is written."""
  tokens, topk, num_experts, cols = 30, 3, 4, 64
  ids = choose(tokens, topk, num_experts, seed=4)
  plan = experts.sort(torch.from_numpy(ids).cuda(), num_experts)
  pairs = tokens * topk
  x, y = make(tokens, cols, torch.bfloat16, 1), make(pairs, cols,
                                                     torch.bfloat16, 2)
  w = make(tokens, topk, torch.float32, 3).cuda()

  def framed(t, pad, value=7.0):
    buf = torch.full((t.shape[0] + 2, t.shape[1] + 2 * pad), value,
                     dtype=t.dtype, device="cuda")
    view = buf[1:-1, pad:-pad]
    view.copy_(t)
    return buf, view

  plain = (experts.gather(x.cuda(), plan), experts.combine(y.cuda(), plan, w),
           *experts.combine_backward(x.cuda(), y.cuda(), plan, w))
  for pad in (3, 8):
    _, xs = framed(x, pad)
    _, ys = framed(y, pad)
    b0, o0 = framed(y, pad)
    b1, o1 = framed(x, pad)
    b2, o2 = framed(y, pad)
    experts.gather(xs, plan, o0)
    experts.combine(ys, plan, w, o1)
    _, gw = experts.combine_backward(xs, ys, plan, w, o2)
    for got, want in ((o0, plain[0]), (o1, plain[1]), (o2, plain[2])):
      assert torch.equal(got, want)
    np.testing.assert_allclose(gw.cpu().numpy(), plain[3].cpu().numpy(),
                               rtol=0, atol=64 * 2 * 2.0 ** -24 * 400)
    for buf, view in ((b0, o0), (b1, o1), (b2, o2)):
      view.fill_(7.0)
      assert bool((buf == 7.0).all())


LAYERS = [  # tokens, topk, experts, in, out
    (1, 1, 1, 32, 16), (4, 2, 8, 64, 128), (64, 4, 16, 256, 200),
    (40, 2, 3, 479, 64), (300, 4, 4, 512, 256), (200, 8, 64, 100, 130),
    (1500, 2, 6, 320, 128), (2, 1, 256, 700, 40), (600, 1, 1, 96, 96),
    (900, 2, 5, 1600, 270), (700, 1, 2, 2048, 128), (30, 2, 40, 9000, 140),
    (100, 40, 50, 160, 64)]


def expert_reference(x_rows, offsets, w, bias, act):
  """The layer over sorted rows of each expert, and its magnitudes."""
  out = w.shape[1]
  y, size = np.zeros((x_rows.shape[0], out)), np.zeros((x_rows.shape[0], out))
  for e in range(w.shape[0]):
    mine = slice(offsets[e], offsets[e + 1])
    if offsets[e] < offsets[e + 1]:
      y[mine], size[mine] = ref.linear(x_rows[mine], w[e],
                                       None if bias is None else bias[e], act)
  return y, size


def expert_weights(mx, num_experts, out, cols, seed=0):
  gen = torch.Generator().manual_seed(seed + num_experts + out + cols)
  w = torch.randn((num_experts, out, cols), generator=gen) * cols ** -0.5
  values = np.stack([ref.quantized(g.double().numpy()) for g in w])
  return mx.quantize(w.cuda()), values


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens,topk,num_experts,cols,out", LAYERS)
def test_linear(mx, experts, tokens, topk, num_experts, cols, out, dtype):
  ids = choose(tokens, topk, num_experts, seed=5)
  plan = experts.sort(torch.from_numpy(ids).cuda(), num_experts)
  offsets, order, _ = ref.sort(ids, num_experts)
  w, values = expert_weights(mx, num_experts, out, cols)
  gen = torch.Generator().manual_seed(out)
  bias = torch.randn((num_experts, out), generator=gen)
  x = make(tokens, cols, dtype, 1)
  sorted_x = x[torch.from_numpy(np.maximum(order, 0) // topk)]
  sorted_x[torch.from_numpy(order < 0)] = float("nan")  # not read
  for b, act, rows, flag in ((None, 0, x, False), (bias, 1, x, False),
                             (bias, 2, sorted_x, True)):
    y = experts.linear(rows.cuda(), plan, w, None if b is None else b.cuda(),
                       act, sorted_rows=flag)
    assert y.dtype == dtype and y.shape == (tokens * topk, out)
    want, size = expert_reference(
        np.nan_to_num(sorted_x.double().numpy()), offsets, values,
        None if b is None else b.double().numpy(), act)
    bound = ref.linear_tolerance(want, size, cols, EPS[dtype])
    assert (np.abs(y.double().cpu().numpy() - want) <= bound).all()
    assert bool((y[offsets[-1]:] == 0).all())
  mx.check()


@pytest.mark.parametrize("cols", [128, 1536])
def test_linear_with_even_and_extreme_groups(mx, experts, cols):
  """All rows in one expert, none at all, and counts around a tile's rows."""
  num_experts, out = 8, 96
  w, values = expert_weights(mx, num_experts, out, cols)
  for counts in ([0, 0, 0, 500, 0, 0, 0, 0], [0] * 8,
                 [127, 128, 129, 1, 0, 255, 256, 257],
                 [15, 16, 17, 1, 0, 31, 32, 33], [1] * 8,
                 [255, 256, 257, 1, 0, 511, 512, 600]):
    ids = np.repeat(np.arange(8), counts)[:, None]
    ids = np.concatenate([ids, np.full((3, 1), -1)])
    np.random.default_rng(1).shuffle(ids)
    plan = experts.sort(torch.from_numpy(ids).cuda(), num_experts)
    offsets, order, _ = ref.sort(ids, num_experts)
    x = make(ids.shape[0], cols, torch.float32, 3)
    y = experts.linear(x.cuda(), plan, w)
    want, size = expert_reference(x.double().numpy()[np.maximum(order, 0)],
                                  offsets, values, None, 0)
    bound = ref.linear_tolerance(want, size, cols, EPS[torch.float32])
    assert (np.abs(y.double().cpu().numpy() - want) <= bound).all()


# tokens, topk, experts, in, out: three tiles or more for every block, in
# uneven groups, for products in tiles of 16, 32, 64 and 128 rows and by pairs
# of blocks.
MANY_TILES = [
    (200, 2, 40, 300, 2000), (500, 2, 40, 300, 2000), (1500, 1, 30, 700, 2000),
    (6000, 2, 20, 300, 1000), (6000, 2, 20, 1600, 1000),
    (6000, 2, 20, 1600, 900)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens,topk,num_experts,cols,out", MANY_TILES)
def test_linear_of_many_tiles(mx, experts, tokens, topk, num_experts, cols, out,
                              dtype):
  """Against 64 bits (summed on the device)."""
  ids = choose(tokens, topk, num_experts, seed=10)
  plan = experts.sort(torch.from_numpy(ids).cuda(), num_experts)
  offsets, order, _ = ref.sort(ids, num_experts)
  w, values = expert_weights(mx, num_experts, out, cols)
  bias = make(num_experts, out, torch.float32, 2)
  x = make(tokens, cols, dtype, 1)
  q = torch.from_numpy(ref.quantized(x.double().numpy())).cuda()
  rows = torch.from_numpy(np.maximum(order, 0) // topk).cuda()
  outputs = [experts.linear(x.cuda(), plan, w, bias.cuda(), mx.ACT_RELU),
             experts.linear(x.cuda()[rows], plan, w, bias.cuda(), mx.ACT_RELU,
                            sorted_rows=True)]
  assert torch.equal(*outputs)
  for e in range(num_experts):
    mine = slice(offsets[e], offsets[e + 1])
    v, b = torch.from_numpy(values[e]).cuda(), bias[e].double().cuda()
    want = torch.relu(q[rows[mine]] @ v.t() + b)
    size = q[rows[mine]].abs() @ v.abs().t() + b.abs()
    bound = (ref.linear_tolerance(0.0, size, cols, EPS[dtype]) +
             EPS[dtype] / 2 * want)
    assert bool(((outputs[0][mine].double() - want).abs() <= bound).all())
  assert bool((outputs[0][offsets[-1]:] == 0).all())
  mx.check()


def mixture(mx, experts, ids, x, w1, b1, w2, b2, weights, num_experts):
  plan = experts.sort(ids, num_experts)
  h = experts.linear(x, plan, w1, b1, mx.ACT_RELU)
  y = experts.linear(h, plan, w2, b2, sorted_rows=True)
  return plan, h, y, experts.combine(y, plan, weights)


@pytest.mark.parametrize("tokens,dtype", [(7, torch.float32),
                                          (500, torch.bfloat16)])
def test_mixture_of_experts(mx, experts, tokens, dtype):
  """Sort, two layers and the way back as they are used together: each step
  against its reference on the step's own inputs, then the whole on a graph
  and on another stream."""
  topk, num_experts, cols, hidden = 3, 5, 160, 224
  ids = choose(tokens, topk, num_experts, seed=6)
  x = make(tokens, cols, dtype, 1).cuda()
  w1, v1 = expert_weights(mx, num_experts, hidden, cols, 1)
  w2, v2 = expert_weights(mx, num_experts, cols, hidden, 2)
  b1 = make(num_experts, hidden, torch.float32, 2).cuda()
  b2 = make(num_experts, cols, torch.float32, 3).cuda()
  weights = torch.softmax(make(tokens, topk, torch.float32, 4), 1).cuda()
  dev = torch.from_numpy(ids).cuda()
  args = (dev, x, w1, b1, w2, b2, weights, num_experts)
  plan, h, y, out = mixture(mx, experts, *args)
  offsets, order, slots = ref.sort(ids, num_experts)
  kept = offsets[-1]
  n = lambda t: t.double().cpu().numpy()  # noqa: E731
  rows = np.where(order[:, None] >= 0, n(x)[order // topk], 0.0)
  for got, (want, size), k in (
      (h, expert_reference(rows, offsets, v1, n(b1), 1), cols),
      (y, expert_reference(n(h), offsets, v2, n(b2), 0), hidden)):
    bound = ref.linear_tolerance(want, size, k, EPS[dtype])
    assert (np.abs(n(got) - want) <= bound)[:kept].all()
  parts = np.where((slots >= 0)[..., None], n(y)[slots], 0.0)
  parts = parts * n(weights)[..., None]
  want = parts.sum(1)
  assert (np.abs(n(out) - want) <= 2 * topk * 2.0 ** -24 *
          np.abs(parts).sum(1) + EPS[dtype] / 2 * np.abs(want)).all()

  stream = torch.cuda.Stream()
  stream.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(stream):
    again = mixture(mx, experts, *args)[-1]
  stream.synchronize()
  assert torch.equal(again, out)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    captured = mixture(mx, experts, *args)[-1]
  captured.zero_()
  graph.replay()
  torch.cuda.synchronize()
  assert torch.equal(captured, out)
  # Other choices in the same buffers: the replay sorts anew.
  dev.copy_(torch.from_numpy(np.roll(ids, 1, axis=0)).cuda())
  graph.replay()
  torch.cuda.synchronize()
  assert torch.equal(captured, mixture(mx, experts, *args)[-1])


def test_empty_batch(mx, experts):
  """No tokens: every call returns its empty outputs."""
  plan = experts.sort(torch.zeros((0, 3), dtype=torch.int64, device="cuda"), 5)
  x = torch.zeros((0, 64), device="cuda")
  w, _ = expert_weights(mx, 5, 32, 64)
  weights = torch.zeros((0, 3), device="cuda")
  assert experts.gather(x, plan).shape == (0, 64)
  assert experts.combine(x, plan, weights).shape == (0, 64)
  assert experts.linear(x, plan, w).shape == (0, 32)
  gy, gw = experts.combine_backward(x, x, plan, weights)
  assert gy.shape == (0, 64) and gw.shape == (0, 3)


@pytest.mark.parametrize("tokens", [6, 200])
def test_rows_off_the_16_byte_grid(mx, experts, tokens):
  """Rows that begin off the grid give the numbers of rows on it."""
  topk, num_experts, cols = 2, 4, 200
  ids = choose(tokens, topk, num_experts, seed=8)
  plan = experts.sort(torch.from_numpy(ids).cuda(), num_experts)
  w, _ = expert_weights(mx, num_experts, 40, cols)
  for dtype in (torch.float32, torch.bfloat16):
    x = make(tokens, cols, dtype, 1).cuda()
    buf = torch.zeros((tokens, cols + 9), dtype=dtype, device="cuda")
    buf[:, 3:3 + cols] = x
    assert torch.equal(experts.linear(buf[:, 3:3 + cols], plan, w),
                       experts.linear(x, plan, w))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cols,pad", [
    (1024, 1), (1025, 0), (1025, 2), (1500, 3), (2047, 4), (2048, 1),
    (2049, 0), (4099, 6)])
@pytest.mark.parametrize("tokens,topk", [(1, 1), (37, 3), (1300, 9)])
def test_gather_long_rows_off_the_grid(experts, tokens, topk, cols, pad,
                                       dtype):
  """Long rows that begin at any element: the bits of x, zeros behind the last
  sorted row, and what lies between the rows of `out` as it was."""
  num_experts = 5
  ids = choose(tokens, topk, num_experts, seed=9)
  plan = experts.sort(torch.from_numpy(ids).cuda(), num_experts)
  order = plan.order.long()
  wide = cols + 2 * pad + 1
  source = make(tokens, wide, dtype, 4).cuda()
  x = source[:, pad:pad + cols]
  store = torch.full((tokens * topk, wide), 7.0, dtype=dtype, device="cuda")
  want = store.clone()
  want[:, pad + 1:pad + 1 + cols] = torch.where(
      (order >= 0)[:, None], x[order.clamp(min=0) // topk], 0.0).to(dtype)
  experts.gather(x, plan, out=store[:, pad + 1:pad + 1 + cols])
  assert torch.equal(store, want)


def test_plan_from_other_tensors(experts):
  """A plan whose arrays lie on no 16-byte boundary, and one sorted into."""
  tokens, topk, num_experts, cols = 50, 4, 6, 64
  ids = torch.from_numpy(choose(tokens, topk, num_experts, seed=7)).cuda()
  plan = experts.sort(ids, num_experts)
  odd = lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)  # noqa: E731
  other = experts.ExpertPlan(odd(plan.offsets), odd(plan.order),
                             odd(plan.slots))
  assert other.slots.data_ptr() % 16 == 4
  y = make(tokens * topk, cols, torch.float32, 1).cuda()
  w = make(tokens, topk, torch.float32, 2).cuda()
  assert torch.equal(experts.combine(y, other, w), experts.combine(y, plan, w))
  other.slots.fill_(-7)
  assert experts.sort(ids, num_experts, other) is other
  for a, b in ((other.offsets, plan.offsets), (other.order, plan.order),
               (other.slots, plan.slots)):
    assert torch.equal(a, b)


def test_offsets_past_32_bits(experts):
  """Sorted rows more than 2^32 bytes apart."""
  tokens, topk, num_experts, cols = 300_000, 8, 16, 1024
  gen = torch.Generator(device="cuda").manual_seed(0)
  ids = torch.randint(0, num_experts, (tokens, topk), generator=gen,
                      device="cuda")
  plan = experts.sort(ids, num_experts)
  x = torch.randint(-8, 8, (tokens, cols), generator=gen, device="cuda",
                    dtype=torch.int8).bfloat16()
  rows = experts.gather(x, plan)
  assert rows.numel() * 2 > 2 ** 32
  some = torch.tensor([0, 1, 77_777, 2_100_000, 2_399_998, 2_399_999],
                      device="cuda")
  assert torch.equal(rows[some], x[plan.order[some].long() // topk])
  back = experts.combine(rows, plan)  # topk times x: exact
  assert torch.equal(back, x * topk)
  gy, gw = experts.combine_backward(x, rows, plan, out_weights(plan))
  assert torch.equal(gy[some], rows[some] * 2)
  want = (x[-5:].double() ** 2).sum(1, keepdim=True).expand(-1, topk)
  assert torch.equal(gw[-5:].double(), want)  # integers below 2^24


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_sort_of_millions(experts, dtype):
  """More than 256 pairs a warp, some dropped: the stable order of torch's
  sort, in which a dropped pair comes last."""
  tokens, topk, num_experts = 300_000, 8, 130
  gen = torch.Generator(device="cuda").manual_seed(1)
  ids = torch.randint(-3, num_experts + 2, (tokens, topk), generator=gen,
                      device="cuda").to(dtype)
  plan = experts.sort(ids, num_experts)
  flat = ids.view(-1).long()
  key = torch.where((flat >= 0) & (flat < num_experts), flat, num_experts)
  by = torch.sort(key, stable=True).indices
  counts = torch.bincount(key, minlength=num_experts + 1)[:num_experts]
  offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
  kept = int(offsets[-1])
  assert kept < flat.numel()
  assert torch.equal(plan.offsets.long(), offsets)
  assert torch.equal(plan.order[:kept].long(), by[:kept])
  assert bool((plan.order[kept:] == -1).all())
  slots = torch.full_like(flat, -1)
  slots[by[:kept]] = torch.arange(kept, device="cuda")
  assert torch.equal(plan.slots.view(-1).long(), slots)


def out_weights(plan):
  return torch.full((plan.tokens, plan.topk), 2.0, device="cuda")


def test_refusals(mx, experts, xse):
  ids = torch.zeros((4, 2), dtype=torch.int32, device="cuda")
  plan = experts.sort(ids, 3)
  x, y = torch.zeros((4, 64), device="cuda"), torch.zeros((8, 64),
                                                          device="cuda")
  weights = torch.zeros((4, 2), device="cuda")
  w = mx.quantize(torch.zeros((3, 32, 64), device="cuda"))
  cases = [
      lambda: experts.sort(ids.float(), 3),
      lambda: experts.sort(ids[0], 3),
      lambda: experts.sort(ids.t(), 3),
      lambda: experts.sort(ids.cpu(), 3),
      lambda: experts.sort(ids, 0),
      lambda: experts.sort(ids, 1025),
      lambda: experts.sort(ids, 4, plan),
      lambda: experts.ExpertPlan(plan.offsets.long(), plan.order, plan.slots),
      lambda: experts.ExpertPlan(plan.offsets, plan.order[:7], plan.slots),
      lambda: experts.gather(y, plan),
      lambda: experts.gather(x.half(), plan),
      lambda: experts.gather(x, plan, x),
      lambda: experts.gather(x, plan, y.bfloat16()),
      lambda: experts.combine(x, plan),
      lambda: experts.combine(y, plan, weights.bfloat16()),
      lambda: experts.combine(y, plan, weights[:3]),
      lambda: experts.combine(y[:, ::2], plan, weights),
      lambda: experts.combine_backward(x.bfloat16(), y, plan, weights),
      lambda: experts.combine_backward(x[:, :32], y, plan, weights),
      lambda: experts.linear(y, plan, w),
      lambda: experts.linear(x, plan, w, sorted_rows=True),
      lambda: experts.linear(x[:, :32], plan, w),
      lambda: experts.linear(x, plan, mx.quantize(torch.zeros(
          (2, 32, 64), device="cuda"))),
      lambda: experts.linear(x, plan, w, torch.zeros(32, device="cuda")),
      lambda: experts.linear(x, plan, w, None, -1),
  ]
  for case in cases:
    with pytest.raises(xse.XseError) as e:
      case()
    assert e.value.code == xse._capi.INVALID_ARGUMENT
