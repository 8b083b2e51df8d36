"""mx.check on the CPU, with a device switch and a library that record: the
failure flag is read on the stream's own device."""

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
