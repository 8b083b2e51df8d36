"""The DLRM tower with 4-bit layers (MATH_MXFP4): every layer against its
64-bit reference on the layer's own input (the tolerance of
mx_reference.linear_tolerance), and the tower through the engine."""

import numpy as np
import pytest
import torch

from tests import mx_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dlrm(xse):
  return xse.dlrm


def check_layers(xse, tower, dense, inter, batch):
  bufs = tower._buffers_for(batch)  # pylint: disable=protected-access
  n = lambda t: t.double().cpu().numpy()  # noqa: E731
  for x, layers, outs in ((dense, tower.bottom, bufs["bottom"]),
                          (inter, tower.top, bufs["top"])):
    for layer, out in zip(layers, outs):
      kernel = n(layer.kernel)
      rows = n(x)[:, :kernel.shape[0]]
      if layer.activation == xse._capi.ACT_SIGMOID:
        want = 1 / (1 + np.exp(-(rows @ kernel + n(layer.bias))))
        np.testing.assert_allclose(n(out), want, rtol=0, atol=1e-5)
      else:
        want, size = ref.linear(rows, ref.quantized(kernel.T), n(layer.bias),
                                layer.activation)
        bound = ref.linear_tolerance(want, size, kernel.shape[0], 2.0 ** -23)
        assert (np.abs(n(out) - want) <= bound).all()
      x = out


@pytest.mark.parametrize("batch", [5, 300])
def test_tower_layers(xse, dlrm, batch):
  tower = dlrm.DenseTower(num_dense=13, num_tables=6, dim=128, seed=3,
                          bottom=(64, 128), top=(96, 40, 1),
                          math=dlrm.MATH_MXFP4)
  gen = torch.Generator().manual_seed(batch)
  dense = torch.randn((batch, 13), generator=gen).cuda()
  pooled = torch.randn((batch, 6, 128), generator=gen).cuda()
  out = tower.forward(dense, pooled)
  assert out.shape == (batch,) and bool(torch.isfinite(out).all())
  check_layers(xse, tower, dense, tower.interaction_rows(batch), batch)
  first = out.clone()
  stream = torch.cuda.Stream()
  stream.wait_stream(torch.cuda.current_stream())
  again = tower.forward(dense, pooled, stream=stream)
  stream.synchronize()
  assert torch.equal(again, first)


@pytest.mark.parametrize("fused", [False, True])
def test_forward_through_the_engine(xse, dlrm, fused):
  batch, tables, dim = 64, 4, 128
  rng = np.random.default_rng(5)
  eng = xse.EmbeddingEngine(0)
  for t in range(tables):
    eng.add_table(f"t{t}", rng.standard_normal((500, dim)).astype(np.float32),
                  "SUM")
    eng.register_feature(f"f{t}", f"t{t}")
  model = dlrm.DLRM(eng, [f"f{t}" for t in range(tables)], dim=dim, seed=1,
                    math=dlrm.MATH_MXFP4, fused_interaction=fused)
  offsets = [torch.arange(0, 3 * batch + 1, 3).cuda() for _ in range(tables)]
  ids = [torch.from_numpy(rng.integers(0, 500, 3 * batch)).cuda()
         for _ in range(tables)]
  dense = torch.from_numpy(rng.standard_normal((batch, 13)).astype(
      np.float32)).cuda()
  out = model.forward(dense, ids, offsets)
  torch.cuda.synchronize()
  assert out.shape == (batch,)
  check_layers(xse, model.tower, dense, model.tower.interaction_rows(batch),
               batch)
  eng.close()
