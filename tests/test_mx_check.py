"""mx.check and its callers on the CPU, with a device switch and a library that
record: the failure flag is read on the stream's own device, and a forward of
4-bit layers reports it where it reports the lookup's errors."""

import contextlib
import types

import pytest
import torch


@pytest.fixture
def calls(xse, monkeypatch):
  """The (device, stream) of each check, and the code that it returns."""
  got = types.SimpleNamespace(seen=[], device=0, rc=xse._capi.OK)

  @contextlib.contextmanager
  def device(d):
    was, got.device = got.device, torch.device(d).index
    yield
    got.device = was

  def check(handle):
    got.seen.append((got.device, handle.value))
    return got.rc

  monkeypatch.setattr(torch.cuda, "device", device)
  monkeypatch.setattr(torch.cuda, "current_stream",
                      lambda: types.SimpleNamespace(cuda_stream=7))
  monkeypatch.setattr(xse._capi.lib, "xse_mxfp4_check", check)
  return got


def stream_of(index, handle):
  return types.SimpleNamespace(device=torch.device("cuda", index),
                               cuda_stream=handle)


def test_check_reads_the_streams_device(xse, calls):
  xse.mx.check(stream_of(1, 11))
  xse.mx.check(stream_of(0, 12))
  xse.mx.check()
  assert calls.seen == [(1, 11), (0, 12), (0, 7)]
  assert calls.device == 0


def test_check_raises(xse, calls):
  calls.rc = xse._capi.DEADLINE_EXCEEDED
  for stream in (None, stream_of(1, 11)):
    with pytest.raises(xse.XseError) as e:
      xse.mx.check(stream)
    assert e.value.code == xse._capi.DEADLINE_EXCEEDED


def forward(xse, monkeypatch, math, fused, status):
  """A DLRM forward whose launches do nothing."""
  engine = types.SimpleNamespace(
      execute_interaction=lambda *args, **kwargs: None,
      execute_batch=lambda *args, **kwargs: None)
  for name in ("bottom_forward", "top_forward", "forward"):
    monkeypatch.setattr(xse.dlrm.DenseTower, name,
                        lambda *args, **kwargs: torch.zeros(3))
  model = xse.dlrm.DLRM(engine, ["a", "b"], dim=128, device="cpu",
                        fused_interaction=fused)
  model.tower.math = math
  model.forward(torch.zeros(3, 13), requests=[], status=status)


@pytest.mark.parametrize("fused", [False, True])
def test_status_of_a_forward_in_4_bits(xse, monkeypatch, calls, fused):
  C, dlrm = xse._capi, xse.dlrm
  found = types.SimpleNamespace(rc=C.OK)
  monkeypatch.setattr(C.lib, "xse_status_create", lambda *args: C.OK)
  monkeypatch.setattr(C.lib, "xse_status_wait", lambda *args: found.rc)
  status = xse.Status()
  stream = stream_of(1, 11)
  calls.rc = C.DEADLINE_EXCEEDED
  forward(xse, monkeypatch, C.MATH_FP32, fused, status)
  status.wait(stream)  # no 4-bit product: nothing to ask
  assert not calls.seen
  forward(xse, monkeypatch, dlrm.MATH_MXFP4, fused, status)
  found.rc = C.INVALID_ARGUMENT  # the lookup's own error comes first
  with pytest.raises(xse.XseError) as e:
    status.wait(stream)
  assert e.value.code == C.INVALID_ARGUMENT and not calls.seen
  found.rc = C.OK
  with pytest.raises(xse.XseError) as e:
    status.wait(stream)
  assert e.value.code == C.DEADLINE_EXCEEDED and calls.seen == [(1, 11)]
  status.wait(stream)  # asked once
  assert calls.seen == [(1, 11)]
