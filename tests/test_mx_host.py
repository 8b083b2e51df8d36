"""Host rules and index arithmetic of the 4-bit and expert kernels at sizes
that are not run on a GPU: a host program over csrc/xse_mx_internal.h."""

import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include "xse_mx_internal.h"

int main(int, char** argv) {
  const long long cols = atoll(argv[1]), size = atoll(argv[2]);
  printf("ring %d\n", xse::ExpertRowFitsRing(cols, size) ? 1 : 0);
  printf("threads %d\n", xse::kRingRowThreads);
  printf("scale %lld\n", static_cast<long long>(
      xse::MxColumnScaleAt(static_cast<int>(cols))));
}
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
  """Runs the host program on some arguments, its lines as a dict."""
  folder = tmp_path_factory.mktemp("host")
  source, program = folder / "host.cc", folder / "host"
  source.write_text(PROGRAM)
  subprocess.run(
      ["g++", "-std=c++17", f"-I{CUDA}/include",
       f"-I{ROOT}/xla-serving_b200/csrc", str(source), "-o", str(program),
       "-ldl"], check=True)

  def run(*args):
    out = subprocess.run([str(program), *map(str, args)], check=True,
                         capture_output=True, text=True).stdout
    return {k: int(v) for k, v in (line.split() for line in out.splitlines())}
  return run


def walk_ends(cols, size, threads):
  """Whether a ring kernel's 32-bit byte offset, `threads` pieces of 16 bytes a
  step, passes the end of a row from each thread's last step."""
  row_end, step = cols * size, 16 * threads
  if row_end >= 2 ** 32:
    return False
  first = max(0, -(-(row_end - step) // 16) * 16)
  return all((b + step) % 2 ** 32 >= row_end
             for b in range(first, row_end, 16))


@pytest.mark.parametrize("cols", [
    4, 1024, 2 ** 29, 2 ** 30 - 2048, 2 ** 30 - 1024, 2 ** 30 - 1020,
    2 ** 30 - 128, 2 ** 30 - 124, 2 ** 30 - 4, 2 ** 30])
@pytest.mark.parametrize("size", [2, 4])
def test_ring_rows_end(host, cols, size):
  """Rows whose byte offsets would wrap are not given to the ring kernels (whose
  thread would then never leave its row), those of ordinary widths are."""
  got = host(cols, size)
  if got["ring"]:
    for threads in (1, 32, got["threads"]):
      assert walk_ends(cols, size, threads)
  assert got["ring"] == (cols * size < 2 ** 32 - 4096)
  if not all(walk_ends(cols, size, t) for t in (32, 256)):
    assert not got["ring"]


@pytest.mark.parametrize("col", [
    0, 31, 32, 127, 128, 4096, 2 ** 29 - 1, 2 ** 29, 2 ** 29 + 96,
    2 ** 30 - 1])
def test_scale_of_a_far_column(host, col):
  """The scale's place by the layout of include/xse_mx.h, past 2^31 bytes too."""
  assert host(col, 4)["scale"] == col // 128 * 512 + col // 32 % 4
